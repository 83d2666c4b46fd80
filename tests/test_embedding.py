"""embedding against the formula, bit for bit (one product in float32, one rounding), and its gradient against sums in 64 bits.

A sum of n float32 values in any order is within n 2^-24 of the sum of their magnitudes; the product with the scale adds one rounding, the
output's type half a step of its own.  Sums of small whole numbers are exact and have to be equal."""
import ctypes as C
import math

import pytest
import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
gpu = pytest.mark.gpu


def table(V, K, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn((V, K), generator=gen).to(DTYPES[dtype]).cuda()


def some_tokens(shape, V, seed, outside=True):
    gen = torch.Generator().manual_seed(seed)
    t = torch.randint(0, V, shape, generator=gen)
    if outside and t.numel() > 3:
        t.view(-1)[1], t.view(-1)[-2] = -1, -(1 << 31)
    return t.cuda()


def rows(w, t, scale, dtype, w_scale=None):
    at = t.clamp(min=0, max=w.shape[0] - 1).long()
    x = w[at].float()
    if w.dtype == torch.int8:
        x = x * w_scale[at].unsqueeze(-1)
    elif w.dtype == torch.float8_e4m3fn:
        x = x * w_scale[at // 128].repeat_interleave(128, -1)[..., :w.shape[1]]
    x = x * torch.tensor(scale, dtype=torch.float32)
    x = torch.where((t < 0).unsqueeze(-1), 0.0, torch.where((t >= w.shape[0]).unsqueeze(-1), math.nan, x))
    return x.to(dtype)


def same(a, b):
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(torch.nan_to_num(a, nan=77.0), torch.nan_to_num(b, nan=77.0)) and torch.equal(a.isnan(), b.isnan())


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("M,V,K", [(1, 1, 1), (1, 50, 7), (5, 100, 8), (33, 100, 101), (300, 1000, 256), (65, 500, 2048), (9, 300, 4099), (2, 20, 20000)])
def test_rows(M, V, K, dtype):
    import rapid_sampling_amd as sample
    w, t = table(V, K, dtype, K), some_tokens((M,), V, M)
    for scale in (1.0, math.sqrt(K), -0.3):
        assert same(sample.embedding(t, w, scale), rows(w, t, scale, w.dtype))
    for out in DTYPES.values():
        assert same(sample.embedding(t.int(), w, 0.7, out_dtype=out), rows(w, t, 0.7, out))


@gpu
def test_shapes_strides_and_tokens_outside():
    import rapid_sampling_amd as sample
    w = table(300, 130, "bf16", 1)
    t = some_tokens((4, 6), 300, 2)
    t[1, 1], t[2, 2] = 300, (1 << 40) + 5
    assert same(sample.embedding(t, w), rows(w, t, 1.0, w.dtype))
    for view in (t[:, ::2], t.t(), t[1], t[0, 0], t[:0], t[:1].expand(5, 6)):
        assert same(sample.embedding(view, w), rows(w, view, 1.0, w.dtype)) and sample.embedding(view, w).shape == view.shape + (130,)
    wide = table(300, 400, "f32", 3)
    for view in (wide[:, 3:103], wide[::3, :50], wide[:1].expand(20, 400), wide[:, 7:8]):
        u = some_tokens((11,), view.shape[0], 4)
        assert same(sample.embedding(u, view), rows(view, u, 1.0, torch.float32))


@gpu
@pytest.mark.parametrize("K", [1, 8, 20, 128, 300, 4096])
@pytest.mark.parametrize("out", list(DTYPES))
def test_tables_in_8_bits(K, out):
    import rapid_sampling_amd as sample
    w, t = table(300, K, "f32", K), some_tokens((50,), 300, 5)
    t[3] = 300
    for q, s in (sample.quantize_int8(w), sample.quantize_fp8(w, block_rows=128)):
        for scale in (1.0, 1.7):
            assert same(sample.embedding(t, q, scale, weight_scale=s, out_dtype=DTYPES[out]), rows(q, t, scale, DTYPES[out], s))
        assert sample.embedding(t, q, weight_scale=s).dtype == torch.float32
        last = q[299:, :].clone() if K % 16 == 0 else q[299:]
        s_last = s[299:] if q.dtype == torch.int8 else s[2:]
        assert same(sample.embedding(t[:1] * 0, last, weight_scale=s_last), rows(last, t[:1] * 0, 1.0, torch.float32, s_last))


def gradient(w, t, g, scale, out_dtype=None):
    import rapid_sampling_amd as sample
    w = w.detach().requires_grad_()
    y = sample.embedding(t, w, scale, out_dtype=out_dtype)
    return torch.autograd.grad(y, w, g)[0]


def check_gradient(w, t, g, scale, got):
    V, K = w.shape
    at = torch.where((t < 0) | (t >= V), V, t).reshape(-1).cpu()
    flat = g.reshape(-1, K).cpu().double()
    sums, sizes = torch.zeros((V + 1, K), dtype=torch.float64), torch.zeros((V + 1, K), dtype=torch.float64)
    sums.index_add_(0, at, flat)
    sizes.index_add_(0, at, flat.abs())
    n = torch.bincount(at, minlength=V + 1).double()[:, None]
    scale32 = float(torch.tensor(scale, dtype=torch.float32))
    want = (sums * scale32)[:-1]
    bound = (2.0 ** -24 * (n + 2) * sizes * abs(scale32))[:-1] + UNIT[w.dtype] * want.abs() * 1.01 + (2.0 ** -25 if w.dtype == torch.float16 else 2.0 ** -149)
    off = (got.cpu().double() - want).abs()
    assert got.dtype == w.dtype and got.shape == w.shape and (off <= bound).all(), (off / bound).max().item()
    assert (got.cpu()[(n[:-1] == 0)[:, 0]] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("M,V,K", [(1, 1, 1), (2, 50, 7), (33, 15, 8), (100, 16, 129), (700, 5, 300), (5000, 3000, 64), (16384, 2047, 12), (16385, 2048, 12), (20000, 70000, 9),
                                   (8193 * 2, 40, 2050), (8192, 300, 5), (8193, 300, 5), (4097, 300, 5)])
def test_gradient(M, V, K, dtype):
    gen = torch.Generator().manual_seed(M + V)
    w, t = table(V, K, dtype, 1), some_tokens((M,), V, M + 7)
    if V > 100:
        t[M // 3: M // 2] = V - 1                                     # one token far more often than the others
        t[M // 2: M // 2 + 40] = V                                    # outside: of no row
    g = torch.randn((M, K), generator=gen).to(w.dtype).cuda()
    got = gradient(w, t, g, 1.3)
    check_gradient(w, t, g, 1.3, got)
    assert torch.equal(got, gradient(w, t.int(), g, 1.3))             # the same again


@gpu
@pytest.mark.parametrize("M", [1, 31, 32, 63, 64, 127, 4096, 16384, 16385, 100000])
@pytest.mark.parametrize("kind", ["one", "last", "none", "two", "each"])
def test_gradient_of_whole_numbers(M, kind):
    """Whole numbers from -3 to 3 are exact in any order, up to 3 * 100000 < 2^24."""
    V, K = 1000, 20
    gen = torch.Generator().manual_seed(M)
    t = {"one": torch.zeros(M), "last": torch.full((M,), V - 1), "none": torch.full((M,), -1), "two": torch.arange(M) // max(1, M // 2) * 500, "each": torch.arange(M) % V}[kind]
    t = t.long().clamp(max=V - 1).cuda()
    g = torch.randint(-3, 4, (M, K), generator=gen).float().cuda()
    got = gradient(torch.zeros((V, K), device="cuda"), t, g, 1.0)
    want = torch.zeros((V + 1, K), dtype=torch.float64)
    want.index_add_(0, torch.where(t < 0, V, t).cpu(), g.cpu().double())
    assert torch.equal(got.cpu().double(), want[:-1])


@gpu
@pytest.mark.parametrize("M", [8192, 8193, 16384, 16385])
def test_gradient_of_whole_numbers_for_a_large_table(M):
    """280 MB of gradient: one workgroup sorts more tokens.  Whole numbers are exact, in bfloat16 up to 256."""
    V, K = 70000, 2000
    gen = torch.Generator().manual_seed(M)
    t = torch.randint(-1, V + 1, (M,), generator=gen)
    t[::100] = 69999
    t, g = t.cuda(), torch.randint(-1, 2, (M, K), generator=gen).bfloat16().cuda()
    got = gradient(torch.zeros((V, K), dtype=torch.bfloat16, device="cuda"), t, g, 1.0)
    there = (t >= 0) & (t < V)
    want = torch.zeros((V, K), device="cuda").index_add_(0, t[there], g[there].float())
    assert want.abs().max() <= 256 and torch.equal(got.float(), want)


@gpu
@pytest.mark.parametrize("V", [1, 2, 2046, 2047, 2048, 131072, 1 << 20, (1 << 22) + 5])
def test_gradient_for_vocabularies_of_any_size(V):
    """One digit of the tokens, two and three."""
    gen = torch.Generator().manual_seed(3)
    for M in (500, 17000):
        t = torch.randint(0, V, (M,), generator=gen).cuda()
        t[:3] = V - 1
        g = torch.randint(-3, 4, (M, 3), generator=gen).float().cuda()
        got = gradient(torch.zeros((V, 3), device="cuda"), t, g, 2.0)
        want = torch.zeros((V, 3), dtype=torch.float64).index_add_(0, t.cpu(), g.cpu().double() * 2)
        assert torch.equal(got.cpu().double(), want)


@gpu
def test_gradients_that_come_in_any_form():
    """Of another type than the table's, broadcast, transposed; tokens of any shape; no token at all."""
    import rapid_sampling_amd as sample
    w, t = table(40, 33, "bf16", 1), some_tokens((5, 7), 40, 2)
    gen = torch.Generator().manual_seed(4)
    g = torch.randn((5, 7, 33), generator=gen).cuda()
    check_gradient(w, t, g, 0.5, gradient(w, t, g, 0.5, torch.float32))
    check_gradient(w, t, g.half(), 0.5, gradient(w, t, g.half(), 0.5, torch.float16))
    f = w.float()
    check_gradient(f, t, g.bfloat16(), 1.0, gradient(f, t, g.bfloat16(), 1.0, torch.bfloat16))
    one = torch.ones((), device="cuda")
    check_gradient(f, t, one.expand(5, 7, 33), 1.0, gradient(f, t, one.expand(5, 7, 33), 1.0))
    row = torch.randn(33, generator=gen).cuda()
    check_gradient(f, t, row.expand(5, 7, 33), 1.0, gradient(f, t, row.expand(5, 7, 33), 1.0))
    turned = torch.randn((33, 7, 5), generator=gen).cuda().permute(2, 1, 0)
    check_gradient(f, t, turned, 1.0, gradient(f, t, turned, 1.0))
    f.requires_grad_()
    sample.embedding(t, f).sum().backward()
    check_gradient(f, t, one.expand(5, 7, 33), 1.0, f.grad)
    assert (gradient(f, t[:0], torch.zeros((0, 7, 33), device="cuda"), 1.0) == 0).all()
    assert torch.equal(gradient(f[:1], t[0, 0] * 0, row, 1.0)[0], row)


@gpu
def test_gradient_against_differences():
    """The table's entries moved one at a time: the sum of g y is linear, so the difference is its derivative up to rounding (2^-22 of 20 terms below 4)."""
    import rapid_sampling_amd as sample
    w = table(6, 5, "f32", 1)
    t = torch.tensor([0, 3, 3, -1, 5, 3, 0], device="cuda")
    g = torch.randn((7, 5), generator=torch.Generator().manual_seed(2)).cuda()
    got = gradient(w, t, g, 1.5)
    for v in range(6):
        for k in range(5):
            up, down = w.clone(), w.clone()
            up[v, k] += 0.5
            down[v, k] -= 0.5
            f = [(sample.embedding(t, x, 1.5).double() * g.double()).sum() for x in (up, down)]
            assert abs((f[0] - f[1]).item() - got[v, k].item()) < 20 * 4 * 4 * 2.0 ** -22


@gpu
def test_more_elements_than_32_bits_count():
    import rapid_sampling_amd as sample
    V, K = 1100000, 2048
    w = torch.zeros((V, K), dtype=torch.bfloat16, device="cuda")
    w[-3:] = table(3, K, "bf16", 1)
    t = torch.tensor([V - 1, 5, V - 3, V], device="cuda")
    assert same(sample.embedding(t, w), rows(w, t, 1.0, w.dtype))
    g = torch.ones((4, K), dtype=torch.bfloat16, device="cuda")
    got = gradient(w, t, g, 1.0)
    assert (got[[V - 1, 5, V - 3]] == 1).all() and got.float().sum() == 3 * K
    del w, got
    M = 1100000
    w = table(7, K, "bf16", 2)
    t = torch.arange(M, device="cuda") % 7
    y = sample.embedding(t, w)
    assert torch.equal(y[-7:], w[t[-7:]]) and torch.equal(y[M // 2], w[t[M // 2]])
    del y
    g = torch.ones((M, K), dtype=torch.bfloat16, device="cuda")
    got = gradient(w.float(), t, g, 1.0, torch.bfloat16)
    assert torch.equal(got[:, 0].cpu(), torch.bincount(t.cpu()).float()) and (got == got[:, :1]).all()


@gpu
def test_from_a_graph_and_on_another_stream():
    import rapid_sampling_amd as sample
    w = table(900, 65, "f32", 1).requires_grad_()
    t = some_tokens((17000,), 900, 2)
    g = torch.randn((17000, 65), generator=torch.Generator().manual_seed(1)).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        held_t = t.clone()
        for _ in range(2):
            y = sample.embedding(held_t, w, 2.0)
            torch.autograd.grad(y, w, g)
        del y
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = sample.embedding(held_t, w, 2.0)
            grad, = torch.autograd.grad(y, w, g)
    for seed in range(3):
        held_t.copy_(some_tokens((17000,), 900, 50 + seed))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, sample.embedding(held_t, w, 2.0)) and torch.equal(grad, gradient(w, held_t, g, 2.0)), seed


def test_refusals():
    import rapid_sampling_amd as sample
    t, w = torch.zeros(3, dtype=torch.long), torch.zeros((4, 16))
    q, s = torch.zeros((4, 16), dtype=torch.int8), torch.ones(4)
    for args, kw, text in [((t.float(), w), {}, "tokens"), ((t, w.double()), {}, "weight"), ((t, w[0]), {}, "shape"), ((t, w), {"out_dtype": torch.float64}, "out_dtype"),
                           ((t, w), {"weight_scale": s}, "weight_scale"), ((t, q), {}, "weight_scale"), ((t, w, math.inf), {}, "finite"), ((t, w), {}, "GPU"),
                           ((t, q), {"weight_scale": s.clone().requires_grad_()}, "gradient"), ((t, w[:0]), {}, "shape")]:
        with pytest.raises(ValueError, match=text):
            sample.embedding(*args, **kw)


@gpu
def test_refusals_on_the_gpu():
    import rapid_sampling_amd as sample
    t, w = torch.zeros(3, dtype=torch.long, device="cuda"), torch.zeros((4, 20), device="cuda")
    q, s = sample.quantize_int8(w)
    f, fs = sample.quantize_fp8(w, block_rows=128)
    for args, kw, text in [((t.cpu(), w), {}, "GPU"), ((t, w.t()), {}, "contiguous"), ((t, q.contiguous()), {"weight_scale": s}, "16 bytes"), ((t, q), {"weight_scale": fs}, "weight_scale"),
                           ((t, f), {"weight_scale": s}, "weight_scale"), ((t, q), {"weight_scale": s[:3]}, "weight_scale")]:
        with pytest.raises(ValueError, match=text):
            sample.embedding(*args, **kw)


def test_refusals_of_the_c_abi():
    from tests import capi
    L = capi.lib()
    p, i32, i64, d, size = C.c_void_p, C.c_int32, C.c_int64, C.c_double, C.c_size_t
    L.rs_embedding.argtypes = [p, i32, i64, p, i32, i64, p, d, i32, i32, i32, p, i32, p]
    L.rs_embedding_workspace_bytes.restype = size
    L.rs_embedding_backward.argtypes = [p, i32, i64, p, i32, i64, d, i32, i32, i32, p, i32, p, size, p]

    def forward(t=256, t64=1, w=256, dtype=0, stride=20, ws=None, M=2, V=5, K=20, y=256, y_dtype=0):
        return L.rs_embedding(t, t64, 1, w, dtype, stride, ws, 1.0, M, V, K, y, y_dtype, None)
    assert forward(t=None) == forward(w=None) == forward(y=None) == forward(dtype=3) == forward(dtype=4) == -4
    assert forward(dtype=5) == forward(y_dtype=3) == forward(t64=2) == -7
    assert forward(M=0) == forward(V=0) == forward(K=0) == forward(M=1 << 24) == forward(stride=-1) == forward(dtype=3, ws=256, stride=16) == -12
    assert forward(t=260) == forward(y=258) == forward(w=258) == forward(dtype=3, ws=256, stride=24) == forward(dtype=4, ws=256, stride=32, w=264) == forward(dtype=3, ws=258, stride=32) == -6
    n = L.rs_embedding_workspace_bytes(2, 5, 20)
    assert n > 0 and L.rs_embedding_workspace_bytes(0, 5, 20) == 0

    def backward(t=256, t64=0, g=256, g_dtype=0, stride=20, M=2, V=5, K=20, dw=256, dtype=0, ws=256, bytes=n):
        return L.rs_embedding_backward(t, t64, 1, g, g_dtype, stride, 1.0, M, V, K, dw, dtype, ws, bytes, None)
    assert backward(t=None) == backward(g=None) == backward(dw=None) == backward(ws=None) == -4
    assert backward(g_dtype=3) == backward(dtype=-1) == backward(t64=3) == -7
    assert backward(M=0) == backward(V=0) == backward(K=0) == backward(M=1 << 24) == backward(stride=-1) == -12
    assert backward(t=258) == backward(g=258) == backward(dw=257, dtype=1) == -6 and backward(bytes=n - 1) == backward(ws=264) == -5
