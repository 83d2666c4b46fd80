"""quantize_fp8 and linear_fp8 against the formulas: the values in 8 bits bit for bit, the product in 64 bits.

With eps = 2^-24 a block's sum of 128 products is within 128 eps of the sum of their magnitudes, the scales and the sums over the
blocks add two roundings a block: eps (128 + 2 blocks + 8) sum |x| |w| bounds the error before the one rounding of the output."""
import math

import pytest
import torch

EPS = 2.0 ** -24
F8 = torch.float8_e4m3fn
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
gpu = pytest.mark.gpu


def blocks_of(x, rows):
    R, K = x.shape
    x = torch.nn.functional.pad(x, (0, -K % 128, 0, -R % rows))
    return x.view(-1, rows, x.shape[1] // 128, 128)


def quantized(x, rows):
    R, K = x.shape
    b = blocks_of(x.cpu().float(), rows)
    scale = (b.abs().amax(dim=(1, 3)) * torch.tensor(1.0 / 448.0)).clamp(min=2.0 ** -126)
    q = (b / scale[:, None, :, None]).to(F8)
    return q.view(torch.uint8).view(b.shape[0] * rows, -1)[:R, :K], scale


def values(q, scale, rows):
    R, K = q.shape
    return (blocks_of(q.cpu().float(), rows).double() * scale.cpu().double()[:, None, :, None]).view(-1, -(-K // 128) * 128)[:R, :K]


def make(R, K, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((R, K), generator=gen) * torch.exp(torch.randn((K,), generator=gen))
    return x.to(DTYPES[dtype]).cuda()


CUT = 7 * 2.0 ** -13


def check(y, x, sx, w, sw, out_dtype, cut=0.0):
    a, b = values(x, sx, 1), values(w, sw, 128)
    want, size = a @ b.T, a.abs() @ b.abs().T
    bound = (EPS * (128 + 2 * sx.shape[-1] + 8) + cut) * size + UNIT[out_dtype] * want.abs() * 1.01 + 2.0 ** -25
    off = (y.cpu().double() - want).abs()
    assert y.dtype == out_dtype and (off <= bound).all(), (off / bound).max().item()


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("R,K", [(1, 1), (3, 7), (1, 128), (2, 129), (130, 255), (257, 1000), (300, 4096)])
@pytest.mark.parametrize("rows", [1, 128])
def test_quantize(R, K, dtype, rows):
    import rapid_sampling_amd as sample
    print("quantize", R, K, dtype, rows, flush=True)
    x = make(R, K, dtype, R + K)
    x[0, :] = 0.0                                                   # a block of nothing
    if R > 1:
        x[1, 0] = 1e-30 if dtype != "f16" else 6e-8
    q, scale = sample.quantize_fp8(x, block_rows=rows)
    want, want_scale = quantized(x, rows)
    assert q.dtype == F8 and q.shape == x.shape and q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0
    assert torch.equal(scale.cpu(), want_scale)
    assert torch.equal(q.view(torch.uint8).cpu(), want)


@gpu
def test_quantize_extremes_and_strides():
    import rapid_sampling_amd as sample
    x = torch.zeros((4, 256), device="cuda")
    x[0, 0], x[0, 1] = 3.4e38, -3.4e38
    x[1, 0], x[1, 1] = 1e-45, -3e-39                                # below the least scale
    x[2, 5] = math.nan
    x[3, 200] = math.inf
    q, scale = sample.quantize_fp8(x)
    want, want_scale = quantized(x, 1)
    assert torch.equal(q[:2].view(torch.uint8).cpu(), want[:2]) and torch.equal(scale[:2].cpu(), want_scale[:2])
    f = q.float()
    assert f[2, 5].isnan() and f[3, 200].isnan() and not f[2, :5].isnan().any() and not f[3, :128].isnan().any()
    y = make(10, 700, "bf16", 3)
    for view in (y[::2, 3:500], y[:, 1:2], y.view(2, 5, 700), y[4]):
        q, scale = sample.quantize_fp8(view)
        want, want_scale = quantized(view.reshape(-1, view.shape[-1]), 1)
        assert torch.equal(q.view(torch.uint8).cpu().reshape(want.shape), want) and torch.equal(scale.cpu().reshape(want_scale.shape), want_scale)
    assert sample.quantize_fp8(y[:0])[0].shape == (0, 700)


@gpu
@pytest.mark.parametrize("exponent", [-149, -130, -126, -122, -117, -110, -104, -100, -96, -70, -61, -60, -59, 0, 110])
@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_halfway_between_two_values(exponent, rows):
    """Numbers at, just below and just above a point halfway between two 8-bit values, in blocks of every size: the division's rounding."""
    import rapid_sampling_amd as sample
    gen = torch.Generator().manual_seed(exponent + 200)
    R = 512
    most = (448.0 * (1.0 + torch.rand((R if rows == 1 else R // 128, 1), generator=gen, dtype=torch.float64)) * 2.0 ** exponent).float()
    most = most.repeat_interleave(rows, 0)
    scale = (most * torch.tensor(1.0 / 448.0)).clamp(min=2.0 ** -126)
    eighths = torch.randint(0, 8, (R, 128), generator=gen).double()
    binade = torch.randint(-6, 8, (R, 128), generator=gen).double()
    half = torch.where(torch.rand((R, 128), generator=gen) < 0.2, (2 * eighths + 1) * 2.0 ** -10, (1 + (2 * eighths + 1) / 16) * 2.0 ** binade)
    x = (half * scale.double()).float()
    x = (x.view(torch.int32) + torch.randint(-2, 3, (R, 128), generator=gen, dtype=torch.int32)).clamp(min=0).view(torch.float32)
    x = torch.minimum(x, most) * torch.where(torch.rand((R, 128), generator=gen) < 0.5, 1.0, -1.0)
    x[:, 0] = most[:, 0]
    q, got_scale = sample.quantize_fp8(x.cuda(), block_rows=rows)
    want, want_scale = quantized(x, rows)
    assert torch.equal(got_scale.cpu(), want_scale)
    off = q.view(torch.uint8).cpu() != want
    assert not off.any(), (off.float().mean().item(), x[off][:4].tolist())


@gpu
@pytest.mark.parametrize("M,K,N", [(1, 16, 1), (1, 100, 50), (2, 128, 16), (1, 4096, 1000), (4, 8192, 70), (3, 8200, 40), (4, 1999, 9000), (5, 1000, 257), (16, 512, 384), (17, 256, 129), (33, 2000, 515),
                                   (64, 144, 640), (77, 2000, 1037), (128, 1024, 256), (129, 128, 128), (257, 300, 700), (512, 2048, 1024), (300, 1, 5)])
@pytest.mark.parametrize("out", list(DTYPES))
def test_product(M, K, N, out):
    import rapid_sampling_amd as sample
    print("product", M, K, N, out, flush=True)
    x, w = make(M, K, "bf16", M), make(N, K, "f32", N)
    qw, sw = sample.quantize_fp8(w, block_rows=128)
    qx, sx = sample.quantize_fp8(x)
    y = sample.linear_fp8(qx, qw, sw, x_scale=sx, out_dtype=DTYPES[out])
    check(y, qx, sx, qw, sw, DTYPES[out], CUT if M > 64 and out != "f32" else 0.0)
    assert torch.equal(y, sample.linear_fp8(x, qw, sw, out_dtype=DTYPES[out]))      # quantised within the call: the same


@gpu
@pytest.mark.parametrize("M", [1, 3, 40, 200])
def test_shapes_types_and_what_lies_behind_the_columns(M):
    import rapid_sampling_amd as sample
    K, N = 200, 300
    store = torch.full((N, 256), 0x7F, dtype=torch.uint8, device="cuda")             # NaN behind every row
    w = make(N, K, "f32", 1)
    qw, sw = sample.quantize_fp8(w, block_rows=128)
    store[:, :K] = qw.view(torch.uint8)
    poisoned = store.view(F8)[:, :K]
    for dtype in DTYPES:
        x = make(M, K, dtype, M)
        y = sample.linear_fp8(x, poisoned, sw)
        qx, sx = sample.quantize_fp8(x)
        check(y, qx, sx, qw, sw, torch.float32)
        held = torch.full((M, 208), 0x7F, dtype=torch.uint8, device="cuda")
        held[:, :K] = qx.view(torch.uint8)
        assert torch.equal(y, sample.linear_fp8(held.view(F8)[:, :K], poisoned, sw, x_scale=sx))
    z = sample.linear_fp8(x.view(1, M, K), qw, sw)
    assert z.shape == (1, M, N) and torch.equal(z[0], sample.linear_fp8(x, qw, sw))
    assert torch.equal(sample.linear_fp8(x[0], qw, sw), sample.linear_fp8(x[:1], qw, sw)[0])
    assert sample.linear_fp8(x[:0], qw, sw).shape == (0, N)
    wide = torch.zeros((M, 2 * K), dtype=x.dtype, device="cuda")                     # rows apart
    wide[:, 1:K + 1] = x
    assert torch.equal(sample.linear_fp8(wide[:, 1:K + 1], qw, sw), sample.linear_fp8(x, qw, sw))


@gpu
@pytest.mark.parametrize("M", [1, 20, 150])
def test_values_that_are_no_numbers_stay_in_their_row(M):
    import rapid_sampling_amd as sample
    x, w = make(M, 384, "f32", 9), make(260, 384, "f32", 10)
    qw, sw = sample.quantize_fp8(w, block_rows=128)
    want = sample.linear_fp8(x, qw, sw)
    x[M // 2, 200] = math.inf
    y = sample.linear_fp8(x, qw, sw)
    assert y[M // 2].isnan().all()
    rest = torch.arange(M, device="cuda") != M // 2
    assert torch.equal(y[rest], want[rest])


@gpu
def test_gradient_of_x_by_the_transposed_weight():
    """d/dx of sum g y is g W, the same product with W's blocks transposed."""
    import rapid_sampling_amd as sample
    w = make(640, 384, "f32", 1)
    qw, sw = sample.quantize_fp8(w, block_rows=128)
    g = make(30, 640, "f32", 2)
    qt, st = qw.t().contiguous(), sw.t().contiguous()
    back = sample.linear_fp8(g, qt, st)
    qg, sg = sample.quantize_fp8(g)
    check(back, qg, sg, qt, st, torch.float32)
    assert torch.equal(values(qt, st, 128), values(qw, sw, 128).T)


@gpu
@pytest.mark.parametrize("N,K", [(515, 384), (1037, 200), (640, 7)])
def test_gradient_of_x_as_it_is_documented(N, K):
    """The module's own lines, for numbers of columns that are no multiples of 16 among others, against g W in 64 bits of the rounded g."""
    import re
    import textwrap

    import rapid_sampling_amd as sample
    lines = re.search(r"\n((?:    .*\n)+?    grad_x = .*\n)", sample.__doc__).group(1)
    weight, weight_scale = sample.quantize_fp8(make(N, K, "f32", 1), block_rows=128)
    grad = make(30, N, "bf16", 2)
    names = {"torch": torch, "sample": sample, "weight": weight, "weight_scale": weight_scale, "grad": grad}
    exec(textwrap.dedent(lines), names)
    qg, sg = sample.quantize_fp8(grad)
    a, b = values(qg, sg, 1), values(weight, weight_scale, 128)
    want, size = a @ b, a.abs() @ b.abs()
    off = (names["grad_x"].cpu().double() - want).abs()
    assert (off <= EPS * (128 + 2 * sg.shape[-1] + 8) * size + 2.0 ** -25).all()


@gpu
def test_head_sampler_and_logprobs_together():
    """hidden states -> logits -> a token each -> its log probability, on another stream and from a graph."""
    import rapid_sampling_amd as sample
    V, K, B = 4096, 512, 6
    qw, sw = sample.quantize_fp8(make(V, K, "f32", 1), block_rows=128)
    u = torch.linspace(0.1, 0.9, B, device="cuda")
    states = sample.setup_rand(0, B)

    def step(hidden):
        logits = sample.linear_fp8(hidden, qw, sw)
        tokens = sample.batch_sampling_temperature_topk_topp(logits, states, 0.9, 5, 1.0, uniforms=u)
        return (logits, tokens) + tuple(sample.token_logprobs(logits, tokens, 0.9, top=5))
    hidden = make(B, K, "bf16", 2)
    logits, tokens, lp, entropy, rank, top_lp, top_tokens = step(hidden)
    assert (rank <= 5).all() and (rank >= 1).all()
    at = (rank.long() - 1)[:, None]
    assert torch.equal(top_tokens.gather(1, at)[:, 0], tokens) and torch.equal(top_lp.gather(1, at)[:, 0], lp)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sample.reserve_workspace(B, V)
        held_in = hidden.clone()
        step(held_in)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step(held_in)
    for seed in range(3):
        fresh = make(B, K, "bf16", 50 + seed)
        held_in.copy_(fresh)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step(fresh))), seed


@gpu
def test_more_elements_than_32_bits_count():
    """The last rows of more than 2^31 outputs, and the last columns of more than 2^31 weights, against parts by themselves."""
    import rapid_sampling_amd as sample
    x, w = make(34000, 128, "bf16", 1), make(65536, 128, "f32", 2)
    qw, sw = sample.quantize_fp8(w, block_rows=128)
    y = sample.linear_fp8(x, qw, sw, out_dtype=torch.bfloat16)
    assert torch.equal(y[-200:], sample.linear_fp8(x[-200:], qw, sw, out_dtype=torch.bfloat16))
    del y
    K, N = 4096, 540000
    store = torch.zeros((N, K), dtype=torch.uint8, device="cuda").view(F8)
    sw = torch.ones(((N + 127) // 128, K // 128), device="cuda")
    x = make(40, K, "bf16", 3)
    store[-256:] = sample.quantize_fp8(make(256, K, "f32", 4), block_rows=128)[0]
    for M in (1, 10, 40):
        y = sample.linear_fp8(x[:M], store, sw)
        qx, sx = sample.quantize_fp8(x[:M])
        part = store[-(256 + N % 128):]
        check(y[:, -part.shape[0]:], qx, sx, part, sw[-3:], torch.float32)
        assert (y[:, :1000] == 0).all()


def test_refusals():
    import rapid_sampling_amd as sample
    x, w, s = torch.zeros((2, 32)), torch.zeros((16, 32), dtype=F8), torch.ones((1, 1))
    bad = [((x, x, s), {}, "float8"), ((x, w[:, :16], s), {}, "K"), ((x, w[0], s), {}, "shape"), ((x, w, s), {"out_dtype": torch.float64}, "out_dtype"),
           ((x, w, s), {}, "GPU")]
    for args, kw, text in bad:
        with pytest.raises(ValueError, match=text):
            sample.linear_fp8(*args, **kw)
    for args, kw, text in [((x.double(),), {}, "float32"), ((x,), {"block_rows": 2}, "block_rows"), ((x[0],), {"block_rows": 128}, "shape"), ((x,), {}, "GPU")]:
        with pytest.raises(ValueError, match=text):
            sample.quantize_fp8(*args, **kw)


@gpu
def test_refusals_on_the_gpu():
    import rapid_sampling_amd as sample
    x, wf = make(2, 100, "f32", 1), make(20, 100, "f32", 2)
    learnt = x.clone().requires_grad_()
    w, s = sample.quantize_fp8(wf, block_rows=128)
    qx, sx = sample.quantize_fp8(x)
    tight = torch.empty(20 * 100, dtype=torch.uint8, device="cuda").view(F8).view(20, 100)      # rows of 100 bytes
    bad = [((x, tight, s), {}, "16 bytes"), ((x, w, s.double()), {}, "weight_scale"), ((x, w, s[:, :0]), {}, "weight_scale"), ((qx, w, s), {}, "x_scale"),
           ((x, w, s), {"x_scale": sx}, "x_scale"), ((qx, w, s), {"x_scale": sx[:1]}, "x_scale"), ((x.t()[:, :2], w[:, :2], s), {}, "contiguous|16 bytes"),
           ((learnt, w, s), {}, "gradient")]
    for args, kw, text in bad:
        with pytest.raises(ValueError, match=text):
            sample.linear_fp8(*args, **kw)
    with pytest.raises(ValueError, match="gradient"):
        sample.quantize_fp8(learnt)
    with torch.no_grad():
        assert sample.linear_fp8(learnt, w, s).shape == (2, 20)


@gpu
def test_scales_without_a_dimension_are_refused():
    """One number for all blocks is no scale for each, not even where there is one block."""
    import rapid_sampling_amd as sample
    x, w = make(1, 100, "f32", 1), make(20, 100, "f32", 2)
    w, s = sample.quantize_fp8(w, block_rows=128)
    qx, sx = sample.quantize_fp8(x)
    with pytest.raises(ValueError, match="weight_scale"):
        sample.linear_fp8(x, w, s[0, 0])
    with pytest.raises(ValueError, match="x_scale"):
        sample.linear_fp8(qx, w, s, x_scale=sx[0, 0])
    assert torch.equal(sample.linear_fp8(qx, w, s, x_scale=sx), sample.linear_fp8(x, w, s))


def test_refusals_of_the_c_abi():
    import ctypes as C

    from tests import capi
    L = capi.lib()
    p, i32, i64 = C.c_void_p, C.c_int32, C.c_int64
    L.rs_quantize_blocks.argtypes = [p, i32, i64, i32, i32, i32, p, i64, p, p]
    L.rs_linear_workspace_bytes.restype = C.c_size_t
    n = L.rs_linear_workspace_bytes()
    L.rs_linear_blocks.argtypes = [p, i64, p, p, i64, p, i32, i32, i32, p, i32, i64, p, C.c_size_t, p]

    def quantize(x=256, dtype=0, rows=1, R=2, K=20, q=256, q_stride=32, scale=256):
        return L.rs_quantize_blocks(x, dtype, K, rows, R, K, q, q_stride, scale, None)
    assert quantize(x=None) == quantize(q=None) == quantize(scale=None) == -4 and quantize(dtype=5) == quantize(rows=64) == -7
    assert quantize(R=0) == quantize(K=0) == quantize(q_stride=16) == -12 and quantize(x=258) == quantize(q=264) == quantize(q_stride=40) == -6

    def linear(x=256, xs=32, w=256, ws=32, sx=256, sw=256, M=2, N=20, K=20, y=256, dtype=0, ys=20, ws_at=256, ws_bytes=n):
        return L.rs_linear_blocks(x, xs, sx, w, ws, sw, M, N, K, y, dtype, ys, ws_at, ws_bytes, None)
    assert linear(x=None) == linear(w=None) == linear(y=None) == linear(sx=None) == linear(sw=None) == linear(ws_at=None) == -4 and linear(dtype=7) == -7
    assert linear(ws_at=264) == linear(ws_bytes=n - 1) == -5
    assert linear(M=0) == linear(N=0) == linear(K=0) == linear(xs=16) == linear(ws=16) == linear(ys=19) == -12
    assert linear(x=264) == linear(w=260) == linear(xs=40) == linear(ws=40) == linear(y=258) == -6

    L.rs_linear_rows.argtypes = [p, i32, i64, p, i64, p, i32, i32, i32, p, i32, i64, p]

    def rows(x=256, dtype=0, w=256, ws=32, sw=256, M=2, N=20, K=20, y=256, y_dtype=0, ys=20):
        return L.rs_linear_rows(x, dtype, K, w, ws, sw, M, N, K, y, y_dtype, ys, None)
    assert rows(x=None) == rows(w=None) == rows(sw=None) == rows(y=None) == -4 and rows(dtype=3) == rows(y_dtype=-1) == -7
    assert rows(M=0) == rows(M=5) == rows(K=8193, ws=8208) == rows(ws=16) == rows(ys=19) == -12 and rows(x=258) == rows(w=260) == rows(ws=40) == -6


@gpu
def test_example():
    """The example runs, and its parts agree: what is scored again is what was answered, up to the logits' rounding to bfloat16
    (2^-9 of logits below 16, twice over: 2^-4 / 0.8 in a log probability), and a row's gradient sums to nothing."""
    import runpy

    from tests.conftest import ROOT
    answers, scored, grad = runpy.run_path(ROOT + "/examples/head_and_logprobs.py")["main"]()
    for step, answer in enumerate(answers):
        assert (answer.logprobs - scored.logprobs[:, step]).abs().max() < 0.1
        assert (answer.top_logprobs[:, :1] >= answer.logprobs[:, None]).all() and (answer.rank <= 50).all()
    assert grad.float().abs().sum() > 0 and grad.float().sum(-1).abs().max() < 1e-3
