"""What a row gives its token is not rounded to 16 bits in the products with G, whatever the number of rows and tokens (from 33 rows on; up to 32, and 64 over
less than sixteen times as many tokens, nothing of G is).  The bounds are those of test_linear_cross_entropy.py, whose sizes are up to 2048 rows of at most a
sixteenth of the vocabulary."""
import pytest
import torch

import tests.test_linear_cross_entropy as base

gpu = pytest.mark.gpu


# tokens of few kinds and of all; vocabularies of one tile and less, and of more than one piece; the rows' order counted and sorted, by one workgroup and by more
@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,V,K,tokens", [(65, 100, 70, 100), (300, 65, 130, 65), (70, 500, 2056, 7), (1286, 1020, 704, 1020), (2048, 3000, 100, 3000), (2048, 33000, 64, 33000), (2049, 33000, 64, 33000),
                                          (2100, 500, 64, 500), (2500, 41000, 24, 60), (4200, 9000, 1040, 9000), (5000, 1, 40, 1), (5000, 2, 300, 2), (8192, 8500, 64, 8500), (8193, 16500, 40, 50),
                                          (9000, 100, 33, 100), (17000, 3000, 40, 3000), (40000, 130, 64, 130)])
def test_many_rows_and_small_vocabularies(M, V, K, tokens, dtype):
    print("tokens", M, V, K, tokens, dtype, flush=True)
    base.test_what_a_row_gives_its_token_is_not_rounded(M, V, K, tokens, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,V,K", [(100, 300, 64), (2300, 700, 72), (9000, 20000, 40)])
def test_rows_without_a_token_and_the_same_again(M, V, K, dtype):
    """Negative tokens and ones outside the vocabulary, a whole batch of them among those; tokens of 32 bits and any distance; the same results every time."""
    x, w, t = base.make(M, V, K, dtype, M)
    gen = torch.Generator().manual_seed(M)
    g, h = torch.rand(M, generator=gen).cuda() / M, torch.randn(M, generator=gen).cuda() * 0.1 / M
    t[::2] = -7
    out, gx, gw = base.gradients(x, w, t, 1.0, g, h)
    f = base.Formula(x, w, t, 1.0)
    f.check(out)
    f.check_gradients(g, h, gx, gw)
    wide = torch.full((M, 3), V - 1, dtype=torch.int32, device="cuda")
    wide[:, 1] = t
    again = base.gradients(x, w, wide[:, 1], 1.0, g, h)
    assert torch.equal(again[1], gx) and torch.equal(again[2], gw)
    none = torch.full_like(t, -1)
    out, gx, gw = base.gradients(x, w, none, 1.0, g, h)
    f = base.Formula(x, w, none, 1.0)
    f.check(out)
    f.check_gradients(g, h, gx, gw)
    t[M // 2] = V
    out, gx, gw = base.gradients(x, w, t, 1.0, g, h)
    rest = torch.arange(M, device="cuda") != M // 2
    assert gx[M // 2].isnan().all() and not gx[rest].isnan().any() and gw.isnan().all()


@gpu
def test_each_gradient_by_itself():
    """Of x alone nothing is put in order; the same numbers."""
    import rapid_sampling_amd as sample
    for M, V, K in ((300, 400, 64), (2500, 3000, 72)):
        x, w, t = base.make(M, V, K, "bf16", 3)
        g = torch.rand(M, generator=torch.Generator().manual_seed(M)).cuda()
        _, gx, gw = base.gradients(x, w, t, 0.9, g)
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(sample.linear_cross_entropy(a, w, t, 0.9).loss, a, g)[0], gx)
        assert torch.equal(torch.autograd.grad(sample.linear_cross_entropy(x, b, t, 0.9).loss, b, g)[0], gw)


@gpu
def test_from_a_graph():
    """More rows than are counted: the sort is captured with the rest."""
    import rapid_sampling_amd as sample
    x, w, t = base.make(9000, 700, 72, "bf16", 2)
    g = torch.rand(9000, generator=torch.Generator().manual_seed(1)).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b, u = x.clone().requires_grad_(), w.clone().requires_grad_(), t.clone()

        def step():
            out = sample.linear_cross_entropy(a, b, u, 0.9)
            return torch.autograd.grad(out.loss, (a, b), g)
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    for seed in range(3):
        fresh, _, tokens = base.make(9000, 700, 72, "bf16", 50 + seed)
        with torch.no_grad():
            a.copy_(fresh)
        u.copy_(tokens)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _, gx, gw = base.gradients(fresh, w, tokens, 0.9, g)
        assert torch.equal(held[0], gx) and torch.equal(held[1], gw), seed
