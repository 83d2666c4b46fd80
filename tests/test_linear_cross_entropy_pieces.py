"""linear_cross_entropy over vocabularies that are worked through in more than one piece: max(8192, 2^27 bytes of G) columns each, so 8192 of 8500 with
8192 rows, 32768 of 33000 with 2048 rows in 16 bits, 16384 in float32.  Bounds as in test_linear_cross_entropy.py, whose formula this is."""
import pytest
import torch

from tests.test_linear_cross_entropy import DTYPES, Formula, gradients, make

gpu = pytest.mark.gpu


def gradients_of(M, seed):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(M, generator=gen) / M).cuda(), (torch.randn(M, generator=gen) * 0.1 / M).cuda()


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("M,V,K", [(8192, 8500, 64), (8192, 8193, 33), (2048, 33000, 64), (2048, 49153, 40), (8192, 16500, 40)])
def test_several_pieces(M, V, K, dtype):
    """Tokens in each piece, at the ends of the pieces among them; each gradient by itself is the same as with the other."""
    import rapid_sampling_amd as sample
    print("pieces", M, V, K, dtype, flush=True)
    x, w, t = make(M, V, K, dtype, M + V)
    t[3], t[4], t[5], t[6] = 8191, 8192, V - 1, -1
    f = Formula(x, w, t, 0.9)
    g, h = gradients_of(M, 5)
    out, gx, gw = gradients(x, w, t, 0.9, g, h)
    f.check(out)
    f.check_gradients(g, h, gx, gw)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = sample.linear_cross_entropy(a, w, t, 0.9)
    assert torch.equal(torch.autograd.grad((out.loss, out.logsumexp), a, (g, h))[0], gx)
    out = sample.linear_cross_entropy(x, b, t, 0.9)
    assert torch.equal(torch.autograd.grad((out.loss, out.logsumexp), b, (g, h))[0], gw)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("first", [0, 8192, 16384])
def test_tokens_of_one_piece_only(first, dtype):
    """All rows' tokens in one piece of three, and few kinds of them."""
    M, V, K = 8192, 16600, 32
    x, w, t = make(M, V, K, dtype, 7)
    t = torch.where(t >= 0, first + t % 60, t)
    f = Formula(x, w, t, 1.0)
    g, h = gradients_of(M, 6)
    out, gx, gw = gradients(x, w, t, 1.0, g, h)
    f.check(out)
    f.check_gradients(g, h, gx, gw)
