"""Rows without a token have no gradient of the loss, whatever stands there: numbers of any size, infinities, NaN.  In float16 G is made as large as
the gradients that count allow, so what is not looked at may not set that factor either.  The same results bit for bit as with zeros there."""
import math

import pytest
import torch

from tests.test_linear_cross_entropy import DTYPES, gradients, make

gpu = pytest.mark.gpu
SIZES = [(7, 500, 40), (20, 131, 2100), (33, 300, 64), (64, 1000, 33), (300, 8000, 72), (1500, 700, 40), (2100, 500, 64), (2500, 41000, 24)]


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("M,V,K", SIZES)
def test_gradients_that_are_not_looked_at(M, V, K, dtype):
    x, w, t = make(M, V, K, dtype, M)
    t[::3] = -1
    gen = torch.Generator().manual_seed(M)
    g, h = torch.rand(M, generator=gen).cuda() * 1e-3, torch.randn(M, generator=gen).cuda() * 1e-4
    g[::3] = 0.0
    for with_h in (None, h):
        want = gradients(x, w, t, 0.8, g, with_h)[1:]
        assert all(v.abs().max() > 0 for v in want)
        for large in (1.0, 1e10, 1e30, -3e38, math.inf, math.nan):
            there = g.clone()
            there[::3] = large
            got = gradients(x, w, t, 0.8, there, with_h)[1:]
            assert all(torch.equal(a, b) for a, b in zip(got, want)), large


@gpu
def test_a_gradient_that_an_infinite_loss_ignores():
    """float16: a row whose logits are all -inf has no gradient; its g, and its h, do not set the factor of the others."""
    x, w, t = make(40, 300, 64, "f16", 4)
    w = -w.abs() - 0.01
    x[5] = math.inf
    g = torch.full((40,), 1e-3, device="cuda")
    h = torch.full((40,), 1e-4, device="cuda")
    g[5], h[5] = 0.0, 0.0
    out, want, _ = gradients(x, w, t, 1.0, g, h)
    assert out.logsumexp[5] == -math.inf and (want[5] == 0).all() and want.abs().max() > 0
    g[5], h[5] = 1e20, -1e25
    assert torch.equal(gradients(x, w, t, 1.0, g, h)[1], want)
