"""linear_cross_entropy and its gradients against the formulas in 64 bits.

With eps = 2^-24: a logit is a float32 sum of K products (each exact, or one rounding for float32 inputs): within d = eps (K + 4) sum |x| |w| / T of its
value, the factor log2(e) / T among them.  lse moves with its logits: d_max, and 2^x, sums of V terms, log2 and the last products add a few roundings of
what they handle: eps (8 + log2-sized numbers).  A sum of V terms in float32: V eps relative, as log: V eps.  The loss is the difference of two such.
A probability is off by 2 d_max + (V + 16) eps of itself; G is rounded to the inputs' type (half a step: UNIT); the products with it are float32 sums
of V or M terms, and rounded once more."""
import ctypes as C
import math

import pytest
import torch

EPS = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -9 * 2, torch.float16: 2.0 ** -12 * 2}
LEAST = {torch.float32: 2.0 ** -140, torch.bfloat16: 2.0 ** -130, torch.float16: 2.0 ** -25}
gpu = pytest.mark.gpu


def make(M, V, K, dtype, seed=1, spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    x, w = torch.randn((M, K), generator=gen), torch.randn((V, K), generator=gen) * (spread / math.sqrt(K))
    t = torch.randint(0, V, (M,), generator=gen)
    if M > 2:
        t[1] = -1
    x = x + 2.0 * w[t.clamp(min=0)]
    return x.to(DTYPES[dtype]).cuda(), w.to(DTYPES[dtype]).cuda(), t.cuda()


class Formula:
    """Everything in 64 bits on the GPU, with how far float32 may be off."""

    def __init__(self, x, w, t, T):
        self.x, self.w, self.T, self.unit, self.least = x.double(), w.double(), T, UNIT[x.dtype], LEAST[x.dtype]
        K, V = x.shape[1], w.shape[0]
        z = self.x @ self.w.t().contiguous() / T
        self.d = (EPS * (K + 4) * (self.x.abs() @ self.w.abs().t().contiguous()) / T).amax(-1)
        self.lse = torch.logsumexp(z, -1)
        self.there = (t >= 0) & (t < V)
        self.at = t.clamp(min=0, max=V - 1)
        self.loss = torch.where(self.there, self.lse - z.gather(1, self.at[:, None])[:, 0], 0.0)
        self.p = torch.exp(z - self.lse[:, None])
        self.d_lse = self.d + EPS * (V + 8 + 4 * self.lse.abs() + 4 * z.abs().amax(-1))
        self.V = V

    def check(self, out):
        for got, want, bound in ((out.logsumexp, self.lse, self.d_lse), (out.loss, self.loss, 2 * self.d_lse)):
            assert got.dtype == torch.float32
            off = (got.double() - want).abs()
            assert (off <= bound).all(), (off / bound).max().item()

    def check_gradients(self, g, h, gx, gw):
        g = torch.where(self.there, g.double(), 0.0)
        h = h.double() if h is not None else torch.zeros_like(g)
        hot = torch.zeros_like(self.p).scatter_(1, self.at[:, None], g[:, None])
        G = ((g + h)[:, None] * self.p - hot) / self.T
        rel = 2 * self.d + EPS * (self.V + 16)
        dG = ((g + h).abs()[:, None] * self.p * rel[:, None] + 4 * EPS * hot.abs()) / self.T + self.unit * G.abs() * 1.01
        if self.unit == UNIT[torch.float16]:
            dG = dG + (g.abs() + h.abs()).max() / self.T * 2.0 ** -38
        dG = dG + LEAST[torch.bfloat16]
        wide = G.abs() + dG
        M, V = G.shape
        for got, want, bound in ((gx, G @ self.w, dG @ self.w.abs() + EPS * (V + 64) * (wide @ self.w.abs())),
                                 (gw, G.t().contiguous() @ self.x, dG.t().contiguous() @ self.x.abs() + EPS * (M + 8) * (wide.t().contiguous() @ self.x.abs()))):
            if got is None:
                continue
            bound = bound + self.unit * want.abs() * 1.01 + self.least
            off = (got.double() - want).abs()
            assert (off <= bound).all(), (off / bound).max().item()


def gradients(x, w, t, T, g, h=None):
    import rapid_sampling_amd as sample
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    out = sample.linear_cross_entropy(x, w, t, T)
    wanted, given = ((out.loss, out.logsumexp), (g, h)) if h is not None else ((out.loss,), (g,))
    return (out,) + torch.autograd.grad(wanted, (x, w), given)


# one row and few, small tiles and large ones, several pieces of the vocabulary, odd sizes of everything
SIZES = [(1, 1, 1), (1, 100, 64), (2, 63, 7), (5, 300, 100), (64, 129, 65), (65, 1000, 33), (130, 700, 130), (200, 5003, 201), (257, 8200, 72), (40, 20011, 64), (1500, 8193, 96), (32, 500, 128), (33, 500, 128), (300, 30011, 24),
         (27, 674, 2100), (155, 556, 1501), (2, 5000, 3000), (300, 65, 1030), (33, 129, 2056), (1, 1, 4000), (32, 1001, 9000), (16, 33001, 100), (9, 300, 5000)]


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("M,V,K", SIZES)
def test_losses_and_gradients(M, V, K, dtype):
    import rapid_sampling_amd as sample
    print("loss", M, V, K, dtype, flush=True)
    for T in (1.0, 0.7):
        x, w, t = make(M, V, K, dtype, M + V)
        f = Formula(x, w, t, T)
        f.check(sample.linear_cross_entropy(x, w, t, T))
        gen = torch.Generator().manual_seed(5)
        g, h = (torch.randn(M, generator=gen) / M).cuda(), (torch.randn(M, generator=gen) * 0.1 / M).cuda()
        out, gx, gw = gradients(x, w, t, T, g, h)
        f.check(out)
        f.check_gradients(g, h, gx, gw)
        again = gradients(x, w, t.int(), T, g, h)
        assert torch.equal(gx, again[1]) and torch.equal(gw, again[2]) and torch.equal(out.loss, again[0].loss)
        _, gx, gw = gradients(x, w, t, T, g)
        f.check_gradients(g, None, gx, gw)


@gpu
@pytest.mark.parametrize("dtype,M,V,K", [("bf16", 2100, 20000, 2048), ("f16", 4200, 9000, 1040), ("f32", 2100, 9000, 1030)])
def test_large_tiles_in_every_product(dtype, M, V, K):
    x, w, t = make(M, V, K, dtype, 3)
    f = Formula(x, w, t, 0.9)
    g = (torch.rand(M, generator=torch.Generator().manual_seed(5)) / M).cuda()
    out, gx, gw = gradients(x, w, t, 0.9, g)
    f.check(out)
    f.check_gradients(g, None, gx, gw)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_shapes_and_strides(dtype):
    """(B, T, K), (K,), no rows; rows at any address and any distance, which are laid out anew, with NaN around them."""
    import rapid_sampling_amd as sample
    x, w, t = make(12, 150, 40, dtype, 1)
    want = sample.linear_cross_entropy(x, w, t)
    Formula(x, w, t, 1.0).check(want)
    g = torch.linspace(-1, 1, 12, device="cuda")
    _, gx, gw = gradients(x, w, t, 1.0, g)
    out, gx3, gw3 = gradients(x.view(3, 4, 40), w, t.view(3, 4), 1.0, g.view(3, 4))
    assert out.loss.shape == (3, 4) and torch.equal(out.loss.view(-1), want.loss) and torch.equal(gx3.view(12, 40), gx) and torch.equal(gw3, gw)
    one = sample.linear_cross_entropy(x[4], w, t[4])
    assert one.loss.shape == () and torch.equal(one.logsumexp, sample.linear_cross_entropy(x[4:5], w, t[4:5]).logsumexp[0])
    out, gx0, gw0 = gradients(x[:0], w, t[:0], 1.0, g[:0])
    assert out.loss.shape == (0,) and gx0.shape == (0, 40) and (gw0 == 0).all()
    for pad, shift in ((40, 8), (41, 0), (43, 3), (64, 1)):
        xs, ws = (torch.full((r, pad + 40), math.nan, dtype=x.dtype, device="cuda")[:, shift:shift + 40] for r in (12, 150))
        xs.copy_(x)
        ws.copy_(w)
        out, gxs, gws = gradients(xs, ws, t, 1.0, g)
        assert torch.equal(out.loss, want.loss) and torch.equal(gxs, gx) and torch.equal(gws, gw)
    wide = torch.full((12, 80), 3, device="cuda")
    wide[:, ::2][:, :1] = t[:, None]
    assert torch.equal(sample.linear_cross_entropy(x, w, wide[:, 0]).loss, want.loss)
    same = x[:1].expand(12, 40)
    assert torch.equal(sample.linear_cross_entropy(same, w, t).logsumexp, sample.linear_cross_entropy(same.contiguous(), w, t).logsumexp)


@gpu
def test_one_gradient_at_a_time_and_broadcast_ones():
    import rapid_sampling_amd as sample
    x, w, t = make(70, 500, 48, "bf16", 2)
    g = torch.full((70,), 1.0 / 70, device="cuda")
    _, gx, gw = gradients(x, w, t, 1.0, g)
    a = x.clone().requires_grad_()
    sample.linear_cross_entropy(a, w, t).loss.mean().backward()
    assert torch.equal(a.grad, gx)
    b = w.clone().requires_grad_()
    sample.linear_cross_entropy(x, b, t).loss.mean().backward()
    assert torch.equal(b.grad, gw)
    a.grad = None
    sample.linear_cross_entropy(a, w, t).logsumexp.sum().backward()
    f = Formula(x, w, t, 1.0)
    f.check_gradients(torch.zeros_like(g), torch.ones_like(g), a.grad, None)
    with torch.no_grad():
        assert not sample.linear_cross_entropy(a, b, t).loss.requires_grad


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,V,K,tokens", [(33, 528, 64, 528), (33, 3001, 100, 5), (64, 1024, 2100, 1024), (64, 900, 70, 900), (50, 130, 2100, 130), (300, 20011, 33, 20011), (300, 4800, 130, 40), (2048, 32768, 64, 32768), (1500, 24000, 1040, 24000), (40, 1048576, 16, 1048576)])
def test_what_a_row_gives_its_token_is_not_rounded(M, V, K, tokens, dtype):
    """From 33 to 2048 rows, of up to a sixteenth of the vocabulary, G's numbers are rounded to 16 bits, but for those at the rows' tokens, which make
    most of a gradient: there the two products hold what the rounding left as well.  (Up to 64 rows over less hold all of it.)  (Tokens of few kinds: rows of dw to which many rows of x give.)"""
    x, w, t = make(M, V, K, dtype, 4, spread=1.0)
    t = torch.where(t >= 0, t * tokens // V * (V // tokens), t)
    t[-1] = V - 1
    gen = torch.Generator().manual_seed(M)
    g, h = torch.randn(M, generator=gen).cuda(), torch.randn(M, generator=gen).cuda() * 0.01
    _, gx, gw = gradients(x, w, t, 0.8, g, h)
    f = Formula(x, w, t, 0.8)
    rows = torch.arange(M, device="cuda")[f.there]
    g = torch.where(f.there, g, 0.0).double()
    hot = torch.zeros_like(f.p).scatter_(1, f.at[:, None], g[:, None])
    G = ((g + h)[:, None] * f.p - hot) / 0.8
    dG = ((g + h).abs()[:, None] * f.p * (2 * f.d + EPS * (V + 16))[:, None] + 4 * EPS * hot.abs()) / 0.8
    rounded = f.unit * G.abs() * 1.01 + (g.abs().max() + h.abs().max()) / 0.8 * 2.0 ** -38
    rounded[rows, f.at[rows]] = 0.0
    dG = dG + rounded + EPS * G.abs() + LEAST[torch.bfloat16]
    wide = G.abs() + dG
    for got, want, bound in ((gx, G @ f.w, dG @ f.w.abs() + EPS * (V + 64) * (wide @ f.w.abs())),
                             (gw, G.t().contiguous() @ f.x, dG.t().contiguous() @ f.x.abs() + EPS * (2 * M + 8) * (wide.t().contiguous() @ f.x.abs()))):
        off, bound = (got.double() - want).abs(), bound + f.unit * want.abs() * 1.01 + f.least
        assert (off <= bound).all(), (off / bound).max().item()


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_gradients_of_sure_tokens_and_rare_ones(dtype):
    """Losses near 0, and tokens of probabilities down to 2^-30, whose rows of w have gradients of that size and no less exact ones."""
    x, w, t = make(64, 400, 128, dtype, 6, spread=1.0)
    x = (x.float() * 0.1 + 14.0 * w[t.clamp(min=0)].float()).to(x.dtype)
    w[300:] *= -1.5
    f = Formula(x, w, t, 1.0)
    g = torch.full((64,), 2.0 ** -16, device="cuda")
    out, gx, gw = gradients(x, w, t, 1.0, g)
    f.check(out)
    f.check_gradients(g, None, gx, gw)
    assert f.loss.min() < 1e-3 and f.p.min() < 2.0 ** -25


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_what_is_no_number_stays_in_its_row(dtype):
    import rapid_sampling_amd as sample
    x, w, t = make(40, 300, 64, dtype, 4)
    want = sample.linear_cross_entropy(x, w, t)
    g = torch.full((40,), 0.1, device="cuda")
    _, gx, _ = gradients(x, w, t, 1.0, g)
    bad = x.clone()
    bad[5, 60], bad[6, 0], bad[7, 63] = math.nan, math.inf, -math.inf
    u = t.clone()
    u[9] = 300
    out, bx, bw = gradients(bad, w, u, 1.0, g)
    rest = torch.ones(40, dtype=torch.bool, device="cuda")
    rest[[5, 6, 7, 9]] = False
    assert out.loss[[5, 6, 7, 9]].isnan().all() and out.logsumexp[[5, 6, 7]].isnan().all() and torch.equal(out.logsumexp[9], want.logsumexp[9])
    assert torch.equal(out.loss[rest], want.loss[rest]) and torch.equal(bx[rest], gx[rest])
    assert bx[[5, 6, 7, 9]].isnan().all() and bw.isnan().all()
    # a token outside the vocabulary has a lse all the same
    a = x.clone().requires_grad_()
    sample.linear_cross_entropy(a, w, u).logsumexp.sum().backward()
    assert not a.grad.isnan().any()


@gpu
def test_rows_of_nothing_but_minus_infinity():
    """Logits that overflow towards -inf all: lse -inf, loss +inf, gradient 0, as token_logprobs has it."""
    import rapid_sampling_amd as sample
    x, w = torch.full((3, 8), 3e38, device="cuda"), torch.full((70, 8), -3e38, device="cuda")
    x[1] = 1e-38
    t = torch.tensor([3, 5, -1], device="cuda")
    out, gx, gw = gradients(x, w, t, 1.0, torch.ones(3, device="cuda"))
    assert out.logsumexp[0] == -math.inf and out.loss[0] == math.inf and out.loss[2] == 0 and out.loss[1].isfinite()
    assert (gx[0] == 0).all() and (gx[2] == 0).all()
    s = sample.token_logprobs(torch.full((1, 70), -math.inf, device="cuda"), t[:1])
    assert s.logprobs[0] == -out.loss[0]


@gpu
@pytest.mark.parametrize("M,V,K,T", [(4, 50, 16, 1.0), (70, 300, 40, 0.7)])
def test_gradients_against_differences(M, V, K, T):
    """Along a direction, in float32: the central difference of the formula in 64 bits at the same points, up to what the two losses may be off, and the
    gradient up to the difference's own error, h^2 / 6 of a third derivative that is at most 4 a^3 for logits that move by a."""
    import rapid_sampling_amd as sample
    x, w, t = make(M, V, K, "f32", 8)
    gen = torch.Generator().manual_seed(9)
    dx, dw = (torch.randn(s.shape, generator=gen).cuda() for s in (x, w))
    dw /= math.sqrt(K)
    g = torch.rand(M, generator=gen).cuda()
    _, gx, gw = gradients(x, w, t, T, g)
    for step_x, step_w in ((dx, 0 * dw), (0 * dx, dw)):
        h = 2.0 ** -7
        ends = [(x + s * h * step_x, w + s * h * step_w) for s in (1, -1)]
        got = [(sample.linear_cross_entropy(a, b, t, T).loss.double() * g).sum().item() for a, b in ends]
        f = [Formula(a, b, t, T) for a, b in ends]
        exact = [(v.loss * g).sum().item() for v in f]
        off = sum((2 * v.d_lse * g).sum().item() for v in f) / (2 * h)
        assert abs((got[0] - got[1]) - (exact[0] - exact[1])) / (2 * h) <= off
        slope = (gx.double() * step_x).sum() + (gw.double() * step_w).sum()
        a = ((step_x.double() @ w.double().t().contiguous() + x.double() @ step_w.double().t().contiguous()) / T).abs().amax(-1)
        rounding = 2.0 ** -20 * ((gx.abs() * step_x.abs()).sum() + (gw.abs() * step_w.abs()).sum()).item()
        assert abs(slope.item() - (exact[0] - exact[1]) / (2 * h)) <= (g * 4 * a ** 3).sum().item() * h * h / 6 + rounding + off


@gpu
def test_against_the_logits_written_out():
    """linear_cross_entropy next to token_logprobs on the logits: -logprob, within the two's bounds, and the same gradients of x."""
    import rapid_sampling_amd as sample
    x, w, t = make(30, 600, 64, "f32", 3)
    out = sample.linear_cross_entropy(x, w, t, 0.8)
    logits = (x.double() @ w.double().t().contiguous()).float()
    lp = sample.token_logprobs(logits, t, 0.8)
    assert (out.loss + lp.logprobs).abs().max() < 2 * Formula(x, w, t, 0.8).d_lse.max() * 2


@gpu
def test_more_elements_than_32_bits_count():
    """The last rows of more than 2^31 weights, and of more than 2^31 activations."""
    import rapid_sampling_amd as sample
    V, K = 600000, 4096
    w = torch.zeros((V, K), dtype=torch.bfloat16, device="cuda")
    x, part, _ = make(20, 300, K, "bf16", 2)
    w[-300:] = part
    t = torch.arange(20, device="cuda") * 7 + V - 300
    out = sample.linear_cross_entropy(x, w, t)
    z = x.double() @ part.double().t().contiguous()
    lse = torch.logsumexp(torch.cat([z, torch.full((20, 1), math.log(V - 300), device="cuda", dtype=torch.float64)], 1), 1)
    assert ((out.logsumexp - lse).abs() < 1e-3).all()
    g = torch.ones(20, device="cuda")
    _, gx, gw = gradients(x, w, t, 1.0, g)
    G = torch.exp(z - lse[:, None])
    G[torch.arange(20), torch.arange(20) * 7] -= 1
    want = G.t().contiguous() @ x.double()
    assert (gw[-300:].double() - want).abs().max() < 2.0 ** -7 * want.abs().max() and gw[: V - 300].abs().max() < 1e-3
    del w, gw
    M = 540000
    x = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda")
    x[-40:] = make(40, 64, K, "bf16", 3)[0]
    w, t = part[:64], torch.arange(M, device="cuda") % 64
    out, gx, gw = gradients(x, w, t, 1.0, torch.ones(M, device="cuda"))
    part_out, px, _ = gradients(x[-256:], w, t[-256:], 1.0, torch.ones(256, device="cuda"))
    # (small tiles there, large ones here: other orders of the sums)
    assert torch.allclose(out.loss[-256:], part_out.loss, rtol=0, atol=1e-3) and (out.loss[:1000] - math.log(64)).abs().max() < 1e-5
    assert (gx[-256:].float() - px.float()).abs().max() <= 2.0 ** -6 * px.float().abs().max()


@gpu
def test_a_tied_table_learns_and_serves():
    """tokens -> embedding -> the same table as the head -> losses, one gradient for both ends; then the table in 8 bits looks up, makes logits,
    and is sampled from.  The gradient is the sum of the two ends' own."""
    import rapid_sampling_amd as sample
    V, K, B, T = 1000, 64, 3, 20
    gen = torch.Generator().manual_seed(1)
    table = (torch.randn((V, K), generator=gen) * 0.3).cuda()
    tokens = torch.randint(0, V, (B, T), generator=gen).cuda()

    def loss_of(lookup, head):
        x = sample.embedding(tokens[:, :-1], lookup, math.sqrt(K))
        return sample.linear_cross_entropy(x, head, tokens[:, 1:]).loss.mean()
    both, lookup, head = (table.clone().requires_grad_() for _ in range(3))
    loss_of(both, both).backward()
    loss_of(lookup, head).backward()
    assert torch.equal(both.grad, lookup.grad + head.grad) or torch.equal(both.grad, head.grad + lookup.grad)
    rows = torch.zeros((V, K), dtype=torch.float64, device="cuda", requires_grad=True)
    w = (table.double() + rows)
    x = w[tokens[:, :-1]] * math.sqrt(K)
    z = x.reshape(-1, K) @ w.t()
    want = (torch.logsumexp(z, -1) - z.gather(1, tokens[:, 1:].reshape(-1, 1))[:, 0]).mean()
    want.backward()
    assert (both.grad - rows.grad).norm() < 1e-5 * rows.grad.norm()
    q, s = sample.quantize_int8(table)
    u = torch.linspace(0.1, 0.9, B, device="cuda")
    states = sample.setup_rand(0, B)
    now = tokens[:, -1]
    for _ in range(3):
        x = sample.embedding(now, q, math.sqrt(K), weight_scale=s, out_dtype=torch.bfloat16)
        logits = sample.linear_int8(x, q, s)
        now = sample.batch_sampling_temperature_topk_topp(logits, states, 1.0, 5, 1.0, uniforms=u)
        answer = sample.token_logprobs(logits, now, top=5)
        assert (answer.rank >= 1).all() and (answer.rank <= 5).all()


@gpu
def test_from_a_graph_and_on_another_stream():
    import rapid_sampling_amd as sample
    x, w, t = make(150, 9000, 72, "bf16", 2)
    g = torch.rand(150, generator=torch.Generator().manual_seed(1)).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()

        def step():
            out = sample.linear_cross_entropy(a, b, t, 0.9)
            return (out.loss, out.logsumexp) + torch.autograd.grad(out.loss, (a, b), g)
        for _ in range(2):
            step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    for seed in range(3):
        fresh = make(150, 9000, 72, "bf16", 50 + seed)[0]
        with torch.no_grad():
            a.copy_(fresh)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        out, gx, gw = gradients(fresh, w, t, 0.9, g)
        assert torch.equal(held[0], out.loss) and torch.equal(held[1], out.logsumexp) and torch.equal(held[2], gx) and torch.equal(held[3], gw), seed


@gpu
def test_derivatives_that_are_refused():
    import torch.autograd.forward_ad as fwd

    import rapid_sampling_amd as sample
    x, w, t = make(6, 50, 16, "f32", 2)
    x.requires_grad_()
    table = w.clone().requires_grad_()
    for value, leaf in ((lambda: sample.linear_cross_entropy(x, w, t).loss.sum(), x), (lambda: sample.linear_cross_entropy(x.detach(), table, t).loss.sum(), table),
                        (lambda: sample.linear_cross_entropy(x, table, t).loss.sum(), table), (lambda: sample.embedding(t, table).square().sum(), table)):
        grad, = torch.autograd.grad(value(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated once"):
            grad.sum().backward()
    with fwd.dual_level():
        dual = fwd.make_dual(w.detach(), torch.ones_like(w))
        for call in (lambda: sample.linear_cross_entropy(dual, w, t[:1].expand(50)), lambda: sample.linear_cross_entropy(x, dual, t), lambda: sample.embedding(t, dual),
                     lambda: sample.quantize_int8(dual), lambda: sample.linear_int8(dual, *sample.quantize_int8(w))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                call()
        out = sample.linear_cross_entropy(x, w, t)
        y = sample.embedding(t, table)
        for value, leaf in ((out.loss, x), (out.logsumexp, x), (y, table)):
            factor = fwd.make_dual(torch.ones_like(value), torch.ones_like(value))
            for again in (False, True):
                with pytest.raises((RuntimeError, ValueError), match="forward-mode"):
                    torch.autograd.grad((value * factor).sum(), leaf, retain_graph=True, create_graph=again)


def test_refusals():
    import rapid_sampling_amd as sample
    x, w, t = torch.zeros((2, 16)), torch.zeros((20, 16)), torch.zeros(2, dtype=torch.long)
    for args, text in [((x.double(), w, t), "float32"), ((x, w.half(), t), "one type"), ((x, w[0], t), "shape"), ((x, w[:, :8], t), "K"), ((x, w, t.float()), "tokens"),
                       ((x, w, t[:1]), "tokens"), ((x, w, t, 0.0), "Temperature"), ((x, w, t, math.nan), "Temperature"), ((x, w, t), "GPU"),
                       ((x, torch.empty((1048577, 16)), t), "Vocabulary"), ((x, w[:0], t), "shape")]:
        with pytest.raises(ValueError, match=text):
            sample.linear_cross_entropy(*args)


@gpu
def test_refusals_on_the_gpu():
    import rapid_sampling_amd as sample
    x, w, t = make(4, 20, 16, "f32")
    for args, text in [((x, w.cpu(), t), "GPU"), ((x, w, t.cpu()), "GPU"), ((x.t().contiguous().t(), w, t), "contiguous"), ((x, w.t().contiguous().t(), t), "contiguous")]:
        with pytest.raises(ValueError, match=text):
            sample.linear_cross_entropy(*args)


def test_refusals_of_the_c_abi():
    from tests import capi
    L = capi.lib()
    p, i32, i64, d, size = C.c_void_p, C.c_int32, C.c_int64, C.c_double, C.c_size_t
    L.rs_lay_out_rows.argtypes = [p, i64, i32, i64, i32, p, i64, p]
    L.rs_linear_cross_entropy_workspace_bytes.restype = size
    L.rs_linear_cross_entropy.argtypes = [p, i64, p, i64, i32, p, i32, i64, i32, i32, i32, d, p, p, p, p, size, p]
    L.rs_linear_cross_entropy_backward.argtypes = [p, i64, p, i64, i32, p, i32, i64, i32, i32, i32, d, p, p, i32, p, i32, p, p, p, size, p]

    def lay(x=256, xs=5, size=2, R=2, K=5, y=256, ys=8):
        return L.rs_lay_out_rows(x, xs, size, R, K, y, ys, None)
    assert lay(x=None) == lay(y=None) == -4 and lay(size=1) == lay(size=8) == -7
    assert lay(R=0) == lay(K=0) == lay(xs=-1) == lay(ys=4) == -12 and lay(x=257) == lay(y=264) == lay(ys=9) == -6
    n = [L.rs_linear_cross_entropy_workspace_bytes(2, 20, 16, 0, b) for b in (0, 1)]
    assert min(n) > 0 and L.rs_linear_cross_entropy_workspace_bytes(0, 20, 16, 0, 0) == L.rs_linear_cross_entropy_workspace_bytes(2, 20, 16, 3, 0) == 0

    def call(back, x=256, xs=16, w=256, ws=16, dtype=0, t=256, t64=1, M=2, V=20, K=16, T=1.0, loss=256, lse=256, stats=256, gs=1, gx=256, gw=256, at=256, bytes=None):
        bytes = n[back] if bytes is None else bytes
        if not back:
            return L.rs_linear_cross_entropy(x, xs, w, ws, dtype, t, t64, 1, M, V, K, T, loss, lse, stats, at, bytes, None)
        return L.rs_linear_cross_entropy_backward(x, xs, w, ws, dtype, t, t64, 1, M, V, K, T, stats, loss, gs, lse, gs, gx, gw, at, bytes, None)
    for b in (0, 1):
        assert call(b, x=None) == call(b, w=None) == call(b, t=None) == call(b, at=None) == -4 and call(b, dtype=3) == call(b, t64=2) == -7
        assert call(b, M=0) == call(b, V=0) == call(b, K=0) == call(b, V=1048577) == call(b, xs=12) == call(b, ws=12) == call(b, xs=1 << 23) == call(b, M=1 << 24, V=1 << 20) == -12
        assert call(b, x=264) == call(b, w=264) == call(b, xs=18) == call(b, ws=17) == call(b, t=260) == call(b, stats=260) == call(b, loss=258) == -6
        assert call(b, T=0.0) == call(b, T=2000.0) == -3 and call(b, at=264) == call(b, bytes=n[b] - 1) == -5
    assert call(0, loss=None) == call(0, lse=None) == call(1, stats=None) == call(1, gx=None, gw=None) == -4
    assert call(1, gs=2) == -7 and call(1, gx=258) == call(1, gw=257, dtype=1) == -6
