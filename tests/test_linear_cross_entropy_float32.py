"""float32 operands of linear_cross_entropy: products of parts in bfloat16 that together are off by a rounding or two, in no direction.

The logsumexp of one logit, or of one that stands far above the others, is that logit, so sums of K products can be read off.  A number x from 1 to 2 is
x0 + r with r < 2^-7; of a product r s is the one part that is rounded before, r and s by 2^-16 at most each: off by 2 * 2^-7 * 2^-16 + 2^-32, so by 4.01 eps of it
(eps = 2^-24).  Up to four products of first parts that one instruction adds are cut off at the last bit of the largest (2 eps of it each, but for that
one); the sum that they come to is cut off at half a step of the result, and theirs with it is rounded (2 eps together); the same of the sums of smaller parts
is below 2^-6 of that.  Together below 6.25 eps sum |x w| + 2 (K - 1) eps max |x w|.
"""
import math

import pytest
import torch

EPS = 2.0 ** -24
gpu = pytest.mark.gpu


def significands(shape, seed):
    """Numbers whose parts are as large as they get (1 + 2^-7 - 2^-23, all ones, ...), and any others; magnitudes from 1 to 2."""
    gen = torch.Generator().manual_seed(seed)
    bits = torch.randint(0, 1 << 23, shape, generator=gen, dtype=torch.int32)
    hard = torch.tensor([0x00FFFF, 0x7FFFFF, 0x00FF7F, 0x017FFF, 0x008000, 0x007FFF, 0x00807F, 0x008080, 0x7F8000, 0x7F7FFF, 0], dtype=torch.int32)
    pick = torch.randint(0, 3 * len(hard), shape, generator=gen)
    bits = torch.where(pick < len(hard), hard[pick.clamp(max=len(hard) - 1)], bits)
    return (bits | 0x3F800000).view(torch.float32)


def logits(x, w):
    """x @ w.T where w has one row, read from the logsumexp."""
    import rapid_sampling_amd as sample
    return sample.linear_cross_entropy(x, w, torch.full((x.shape[0],), -1, device="cuda")).logsumexp


@gpu
@pytest.mark.parametrize("M", [1, 7, 16, 17, 64, 500, 5000])
@pytest.mark.parametrize("K", [1, 2, 3, 4])
def test_products_of_a_few_numbers(M, K):
    for seed in range(8):
        x, w = significands((M, K), seed).cuda(), significands((1, K), 50 + seed).cuda()
        if seed % 2:
            x *= torch.where(torch.rand(x.shape, generator=torch.Generator().manual_seed(seed)) < 0.5, -1.0, 1.0).cuda()
        if seed == 0:
            x[0], w[0] = 1.0 + 2.0 ** -7 - 2.0 ** -23, 1.0 + 2.0 ** -7 - 2.0 ** -23
        for scale in (1.0, 2.0 ** 40, 2.0 ** -40):
            products = x.double() * w.double()
            off = (logits(x * scale, w / scale).double() - products.sum(1)).abs()
            bound = EPS * (6.25 * products.abs().sum(1) + 2 * (K - 1) * products.abs().amax(1))
            assert (off <= bound).all(), (seed, scale, (off / bound).max().item())


@gpu
@pytest.mark.parametrize("M,V", [(300, 300), (2048, 2048), (4096, 4096)])
def test_products_in_tiles_of_every_size(M, V):
    """One logit far above the others, which are some 2^7 below it."""
    K = 3
    x, w = (significands((M, K), 1) * 16.0).cuda(), -significands((V, K), 2).cuda()
    w[V // 2] *= -1.0
    products = x.double() * w[V // 2].double()
    off = (logits(x, w).double() - products.sum(1)).abs()
    assert (off <= EPS * (6.25 * products.sum(1) + 2 * (K - 1) * products.amax(1))).all()


@gpu
@pytest.mark.parametrize("M", [16, 64])
def test_no_direction(M):
    """What a product is off by has no sign of its own.  One step of the sum has: where a larger product comes to a smaller sum, as the two first
    parts' does to those of the others, the matrix instruction cuts the sum off downwards at half a step of the result (2^-23 of it), and so by a
    quarter of one on average: half a unit.  (Measured with 1 and f 2^-23: f of 1, 1.25, 1.5, 1.75 give 1, 1, 2, 2; -0.125 gives what -0.5 does.)  Over 4096
    products, each off by less than 6.25 units and by less than one in the root of the mean square, the mean stays within that and 6 / sqrt(4096).  (With
    the second parts cut off there as well: -0.91.)"""
    off, size = 0.0, 0
    for seed in range(4096 // M):
        gen = torch.Generator().manual_seed(100 + seed)
        x, w = (torch.rand((M, 1), generator=gen) + 1.0).cuda(), (torch.rand((1, 1), generator=gen) + 1.0).cuda()
        want = x.double() @ w.double()
        off += ((logits(x, w).double()[:, None] - want) / want).sum().item()
        size += M
    assert abs(off / size) <= (0.5 + 6.0 / math.sqrt(size)) * EPS


@gpu
def test_the_largest_numbers():
    """Numbers that a rounding to bfloat16 would take to infinity: from 2^128 - 2^119 on."""
    import rapid_sampling_amd as sample
    top = torch.tensor([0x7F7FFFFF, 0x7F7F8000, 0x7F7F7FFF, 0x7F7F0001, 0x7F7F0000], dtype=torch.int32).view(torch.float32)
    for sign in (1.0, -1.0):
        for M in (1, 5, 40, 300):
            x = (sign * top).repeat((M + 4) // 5)[:M, None].cuda()
            small = torch.tensor([[2.0 ** -126 * 1.5]], device="cuda")
            for got, a in ((logits(x, small), x), (logits(small.expand(M, 1), x[:1]), x[:1].expand(M, 1))):
                want = a.double()[:, 0] * small.double()[0, 0]
                assert ((got.double() - want).abs() <= 6.25 * EPS * want.abs()).all()
    x, w = top[:1, None].cuda(), torch.tensor([[1.0], [0.5]], device="cuda")
    out = sample.linear_cross_entropy(x, w, torch.tensor([0], device="cuda"))
    assert out.logsumexp[0].item() == top[0].item() and out.loss[0] == 0


@gpu
@pytest.mark.parametrize("M,V,K", [(5, 40, 33), (60, 200, 100), (300, 700, 64)])
def test_gradients_of_one_sign(M, V, K):
    """Numbers of one sign, so that every error that has a direction adds up: dw's rows are G^T x with x of one sign."""
    from tests.test_linear_cross_entropy import Formula, gradients
    gen = torch.Generator().manual_seed(M)
    x, w = significands((M, K), 3).cuda(), (significands((V, K), 4) / K).cuda()
    t = torch.randint(0, V, (M,), generator=gen).cuda()
    f = Formula(x, w, t, 1.0)
    g = torch.ones(M, device="cuda")
    out, gx, gw = gradients(x, w, t, 1.0, g)
    f.check(out)
    f.check_gradients(g, None, gx, gw)
