"""quantize_int8 and linear_int8 against the formulas, bit for bit: the integers and scales as one division and one rounding give them, the
sums exactly (float64 holds whole numbers up to 2^53), the result as float32(sum) * (x_scale * w_scale) and one rounding to the output's type."""
import ctypes as C
import math

import pytest
import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
gpu = pytest.mark.gpu


def make(R, K, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((R, K), generator=gen) * torch.exp(torch.randn((K,), generator=gen))
    return x.to(DTYPES[dtype]).cuda()


def quantized(x):
    x = x.cpu().float()
    scale = (x.abs().amax(-1) * torch.tensor(1.0 / 127.0)).clamp(min=2.0 ** -126)
    return torch.round(x / scale.unsqueeze(-1)).to(torch.int8), scale


def product(x, sx, w, sw, dtype):
    sums = x.cpu().double() @ w.cpu().double().T
    assert sums.abs().max() < 2 ** 31
    return (sums.float() * (sx.cpu().view(-1, 1) * sw.cpu().view(1, -1))).to(dtype)


def integers(R, K, seed, stride=None):
    """Any integers of 8 bits, -128 among them, and 77 behind the columns."""
    gen = torch.Generator().manual_seed(seed)
    store = torch.full((R, stride or K + -K % 16), 77, dtype=torch.int8)
    store[:, :K] = torch.randint(-128, 128, (R, K), generator=gen)
    return store.cuda()[:, :K]


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("R,K", [(1, 1), (3, 7), (5, 64), (7, 129), (130, 512), (130, 513), (9, 2048), (9, 2049), (3, 8192), (3, 20001)])
def test_quantize(R, K, dtype):
    import rapid_sampling_amd as sample
    x = make(R, K, dtype, R + K)
    x[0] = 0.0
    if R > 1:
        x[1] = x[1] * 0.0 + (6e-8 if dtype == "f16" else 1e-39)             # below the least scale
        x[1, 0] = -x[1, 0]
    q, scale = sample.quantize_int8(x)
    want, want_scale = quantized(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0
    assert torch.equal(scale.cpu(), want_scale) and torch.equal(q.cpu(), want)
    whole = torch.as_strided(q, (R, q.stride(0)), (q.stride(0), 1))
    assert (whole[:, K:] == 0).all()


@gpu
def test_quantize_strides_and_what_is_no_number():
    import rapid_sampling_amd as sample
    y = make(10, 700, "bf16", 3)
    for view in (y[::2, 3:500], y[:, 1:2], y.view(2, 5, 700), y[4], y[:1].expand(6, 700)):
        q, scale = sample.quantize_int8(view)
        want, want_scale = quantized(view)
        assert torch.equal(q.cpu(), want) and torch.equal(scale.cpu(), want_scale) and scale.shape == view.shape[:-1]
    assert sample.quantize_int8(y[:0])[0].shape == (0, 700)
    x = make(4, 3000, "f32", 4)
    keep = quantized(x)
    x[1, 2900], x[2, 5], x[3, 7] = math.nan, math.inf, -math.inf
    q, scale = sample.quantize_int8(x)
    assert scale[1:].isnan().all() and (q[1:] == 0).all() and torch.equal(q[0].cpu(), keep[0][0]) and scale[0].cpu() == keep[1][0]


@gpu
@pytest.mark.parametrize("exponent", [-149, -130, -126, -122, -110, -100, -70, -61, -60, -59, 0, 110])
def test_quantize_halfway_between_two_integers(exponent):
    """Numbers at, just below and just above a point halfway between two integers: the division's rounding."""
    import rapid_sampling_amd as sample
    gen = torch.Generator().manual_seed(exponent + 200)
    most = (127.0 * (1.0 + torch.rand((512, 1), generator=gen, dtype=torch.float64)) * 2.0 ** exponent).float()
    scale = (most * torch.tensor(1.0 / 127.0)).clamp(min=2.0 ** -126)
    half = torch.randint(-127, 127, (512, 128), generator=gen).double() + 0.5
    x = (half * scale.double()).float()
    x = (x.abs().view(torch.int32) + torch.randint(-2, 3, (512, 128), generator=gen, dtype=torch.int32)).clamp(min=0).view(torch.float32) * torch.sign(half).float()
    x = torch.minimum(x.abs(), most) * torch.sign(x)
    x[:, 0] = most[:, 0]
    q, got = sample.quantize_int8(x.cuda())
    want, want_scale = quantized(x)
    assert torch.equal(got.cpu(), want_scale) and torch.equal(q.cpu(), want)


# few rows (one and two rows of w's fragments to a wave), small tiles whole and shared, large tiles; odd sizes of everything
SIZES = [(1, 16, 1), (1, 100, 50), (1, 4096, 9000), (2, 128, 16), (3, 127, 8193), (4, 8192, 70), (16, 1000, 257), (17, 1000, 257), (33, 2000, 515), (64, 144, 640),
         (64, 4100, 130), (77, 2000, 1037), (129, 130, 700), (300, 65, 5), (2000, 200, 6200), (1025, 1029, 10007), (3, 100, 40001), (100, 300, 33000), (300, 77, 40000),
         (64, 8200, 1300), (77, 2000, 5037), (33, 515, 9001), (20, 40001, 1000), (129, 130, 3700), (16, 15000, 7000)]


@gpu
@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("out", list(DTYPES))
def test_product(M, K, N, out):
    import rapid_sampling_amd as sample
    print("product", M, K, N, out, flush=True)
    x, w = integers(M, K, M + K), integers(N, K, N + 1)
    sx, sw = torch.rand(M).cuda() + 0.5, torch.rand(N).cuda() + 0.5
    y = sample.linear_int8(x, w, sw, x_scale=sx, out_dtype=DTYPES[out])
    # (sums up to 2^20 times scales up to 2.25 leave float16, on both sides)
    assert torch.equal(y.cpu(), product(x, sx, w, sw, DTYPES[out]))


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("M,K,N", [(1, 200, 300), (3, 8192, 300), (4, 1000, 20000), (5, 200, 300), (40, 200, 300), (200, 200, 300)])
def test_rounding_within_the_call(M, K, N, dtype):
    import rapid_sampling_amd as sample
    x = make(M, K, dtype, M)
    w, sw = sample.quantize_int8(make(N, K, "f32", N))
    qx, sx = quantized(x)
    want = product(qx, sx, w, sw, torch.float32)
    assert torch.equal(sample.linear_int8(x, w, sw).cpu(), want)
    wide = torch.zeros((M, 2 * K), dtype=x.dtype, device="cuda")                    # rows apart
    wide[:, 1:K + 1] = x
    assert torch.equal(sample.linear_int8(wide[:, 1:K + 1], w, sw).cpu(), want)
    assert torch.equal(sample.linear_int8(x.view(1, M, K), w, sw.view(-1, 1)).cpu()[0], want)
    assert torch.equal(sample.linear_int8(x[0], w, sw).cpu(), want[0])
    given, given_scale = sample.quantize_int8(x[0])
    assert torch.equal(sample.linear_int8(given, w, sw, x_scale=given_scale).cpu(), want[0])
    assert sample.linear_int8(x[:0], w, sw).shape == (0, N)
    same = x[:1].expand(M, K)                                                       # the same row in every place
    assert torch.equal(sample.linear_int8(same, w, sw).cpu(), want[:1].expand(M, N))


@gpu
@pytest.mark.parametrize("M", [1, 17, 130])
def test_the_largest_sums(M):
    """131071 products of -128 with itself: 2^31 - 16384."""
    import rapid_sampling_amd as sample
    K, N = 131071, 131
    x = torch.full((M, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    w = torch.full((N, K + 1), -128, dtype=torch.int8, device="cuda")[:, :K]
    w[1] = 127
    one = torch.ones(max(M, N), device="cuda")
    y = sample.linear_int8(x, w, one[:N], x_scale=one[:M])
    assert (y[:, 0] == float(K * 16384)).all() and (y[:, 1] == torch.tensor(-K * 128 * 127).float().cuda()).all() and (y[:, 2:] == float(K * 16384)).all()
    with pytest.raises(ValueError, match="too large"):
        sample.linear_int8(torch.zeros((1, 131072), dtype=torch.int8, device="cuda"), torch.zeros((1, 131072), dtype=torch.int8, device="cuda"), one[:1], x_scale=one[:1])


@gpu
@pytest.mark.parametrize("M", [1, 4, 20, 150])
def test_values_that_are_no_numbers_stay_in_their_row(M):
    import rapid_sampling_amd as sample
    x = make(M, 384, "f32", 9)
    w, sw = sample.quantize_int8(make(260, 384, "f32", 10))
    want = sample.linear_int8(x, w, sw)
    x[M // 2, 200] = math.inf
    y = sample.linear_int8(x, w, sw)
    rest = torch.arange(M, device="cuda") != M // 2
    assert y[M // 2].isnan().all() and torch.equal(y[rest], want[rest])


@gpu
def test_rows_that_lie_far_apart():
    """More bytes between two rows than 32 bits reach over a tile, and more than 2^31 weights and results."""
    import rapid_sampling_amd as sample
    store = integers(3, 48, 1, stride=1 << 24)
    one = torch.ones(1 << 17, device="cuda")
    x = integers(70, 48, 2)
    y = sample.linear_int8(x, store, one[:3], x_scale=one[:70])
    assert torch.equal(y.cpu(), product(x, one[:70], store, one[:3], torch.float32))
    del store
    M, N, K = 34000, 65536, 128
    x, w = integers(M, K, 3), integers(N, K, 4)
    y = sample.linear_int8(x, w, one[:N], x_scale=one[:M], out_dtype=torch.float16)
    assert torch.equal(y[-200:], sample.linear_int8(x[-200:], w, one[:N], x_scale=one[:200], out_dtype=torch.float16))
    del y
    K, N = 4096, 540000
    store = torch.zeros((N, K), dtype=torch.int8, device="cuda")
    store[-256:] = integers(256, K, 5)
    one = torch.ones(N, device="cuda")
    for M in (1, 40, 300):
        x = integers(M, K, 6)
        y = sample.linear_int8(x, store, one, x_scale=one[:M])
        assert torch.equal(y[:, -256:].cpu(), product(x, one[:M], store[-256:], one[:256], torch.float32)) and (y[:, :1000] == 0).all()


@gpu
def test_from_a_graph_and_on_other_streams():
    """Captured without anything reserved; graphs captured on one stream run side by side on two, each with its own workspace."""
    import rapid_sampling_amd as sample
    from tests.test_operator_workspaces import fresh_stream
    w, sw = sample.quantize_int8(make(1200, 16384, "f32", 1))               # (whose columns are shared out, from 17 rows on)
    inputs = [make(M, 16384, "bf16", M) for M in (2, 40, 100)]
    want = [sample.linear_int8(x, w, sw) for x in inputs]
    torch.cuda.synchronize()
    side, sets = fresh_stream(), []
    with torch.cuda.stream(side):
        for _ in range(2):
            held_in = [x.clone() for x in inputs]
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                held = [sample.linear_int8(x, w, sw) for x in held_in]
            sets.append((graph, held_in, held))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed in range(4):
        for n, (graph, held_in, held) in enumerate(sets):
            for x in held_in:
                x.copy_(make(x.shape[0], 16384, "bf16", 90 + 2 * seed + n))
        torch.cuda.synchronize()
        for stream, (graph, held_in, held) in zip(streams, sets):
            with torch.cuda.stream(stream):
                for _ in range(5):
                    graph.replay()
        torch.cuda.synchronize()
        for graph, held_in, held in sets:
            assert all(torch.equal(y, sample.linear_int8(x, w, sw)) for x, y in zip(held_in, held)), seed
    # products of either kind take turns at one workspace
    w8, s8 = sample.quantize_fp8(make(1200, 16384, "f32", 1), block_rows=128)
    fp8 = sample.linear_fp8(inputs[1], w8, s8)
    for _ in range(5):
        assert torch.equal(sample.linear_int8(inputs[1], w, sw), want[1]) and torch.equal(sample.linear_fp8(inputs[1], w8, s8), fp8)


def test_refusals():
    import rapid_sampling_amd as sample
    x, w, s = torch.zeros((2, 32)), torch.zeros((16, 32), dtype=torch.int8), torch.ones(16)
    for args, kw, text in [((x, x, s), {}, "int8"), ((x, w[:, :16], s), {}, "K"), ((x, w[0], s), {}, "shape"), ((x, w, s), {"out_dtype": torch.float64}, "out_dtype"),
                           ((x, w, s), {}, "GPU"), ((x.clone().requires_grad_(), w, s), {}, "gradient"), ((x, w, s.clone().requires_grad_()), {}, "gradient")]:
        with pytest.raises(ValueError, match=text):
            sample.linear_int8(*args, **kw)
    for args, text in [((x.double(),), "float32"), ((x,), "GPU"), ((x.sum(),), "shape")]:
        with pytest.raises(ValueError, match=text):
            sample.quantize_int8(*args)


@gpu
def test_refusals_on_the_gpu():
    import rapid_sampling_amd as sample
    x = make(2, 100, "f32", 1)
    w, s = sample.quantize_int8(make(20, 100, "f32", 2))
    qx, sx = sample.quantize_int8(x)
    tight = torch.zeros((20, 100), dtype=torch.int8, device="cuda")                 # rows of 100 bytes
    bad = [((x, tight, s), {}, "16 bytes"), ((x, w, s.double()), {}, "weight_scale"), ((x, w, s[:19]), {}, "weight_scale"), ((x, w, s[0]), {}, "weight_scale"),
           ((x, w, s.cpu()), {}, "weight_scale"), ((qx, w, s), {}, "x_scale"), ((x, w, s), {"x_scale": sx}, "x_scale"), ((qx, w, s), {"x_scale": sx[:1]}, "x_scale"),
           ((qx, w, s), {"x_scale": sx.repeat_interleave(2)[::2]}, "x_scale"), ((x.t()[:, :2], w[:, :2], s), {}, "contiguous|16 bytes"),
           ((x.clone().requires_grad_(), w, s), {}, "gradient")]
    for args, kw, text in bad:
        with pytest.raises(ValueError, match=text):
            sample.linear_int8(*args, **kw)
    with pytest.raises(ValueError, match="gradient"):
        sample.quantize_int8(x.clone().requires_grad_())
    with torch.no_grad():
        assert sample.linear_int8(x.clone().requires_grad_(), w, s).shape == (2, 20)


def test_refusals_of_the_c_abi():
    from tests import capi
    L = capi.lib()
    p, i32, i64 = C.c_void_p, C.c_int32, C.c_int64
    L.rs_quantize_rows.argtypes = [p, i32, i64, i32, i32, p, i64, p, p]
    L.rs_linear_workspace_bytes.restype = C.c_size_t
    n = L.rs_linear_workspace_bytes()
    L.rs_linear_int8.argtypes = [p, i64, p, p, i64, p, i32, i32, i32, p, i32, i64, p, C.c_size_t, p]
    L.rs_linear_int8_rows.argtypes = [p, i32, i64, p, i64, p, i32, i32, i32, p, i32, i64, p]

    def quantize(x=256, dtype=0, xs=20, R=2, K=20, q=256, q_stride=32, scale=256):
        return L.rs_quantize_rows(x, dtype, xs, R, K, q, q_stride, scale, None)
    assert quantize(x=None) == quantize(q=None) == quantize(scale=None) == -4 and quantize(dtype=5) == -7
    assert quantize(R=0) == quantize(K=0) == quantize(q_stride=16) == quantize(xs=-1) == quantize(K=1 << 25, q_stride=1 << 25) == -12
    assert quantize(x=258) == quantize(q=264) == quantize(q_stride=40) == quantize(scale=258) == -6

    def linear(x=256, xs=32, w=256, ws=32, sx=256, sw=256, M=2, N=20, K=20, y=256, dtype=0, ys=20, ws_at=256, ws_bytes=n):
        return L.rs_linear_int8(x, xs, sx, w, ws, sw, M, N, K, y, dtype, ys, ws_at, ws_bytes, None)
    assert linear(x=None) == linear(w=None) == linear(y=None) == linear(sx=None) == linear(sw=None) == linear(ws_at=None) == -4 and linear(dtype=7) == -7
    assert linear(ws_at=264) == linear(ws_bytes=n - 1) == -5
    assert linear(M=0) == linear(N=0) == linear(K=0) == linear(xs=16) == linear(ws=16) == linear(ys=19) == linear(K=131072, xs=1 << 18, ws=1 << 18) == -12
    assert linear(M=1 << 24, N=1 << 16, ys=1 << 16) == linear(M=1 << 25) == linear(M=(1 << 19) + 1, ws=1 << 25) == -12
    assert linear(x=264) == linear(w=260) == linear(xs=40) == linear(ws=40) == linear(y=258) == -6

    def rows(x=256, dtype=0, xs=20, w=256, ws=32, sw=256, M=2, N=20, K=20, y=256, y_dtype=0, ys=20):
        return L.rs_linear_int8_rows(x, dtype, xs, w, ws, sw, M, N, K, y, y_dtype, ys, None)
    assert rows(x=None) == rows(w=None) == rows(sw=None) == rows(y=None) == -4 and rows(dtype=3) == rows(y_dtype=-1) == -7
    assert rows(M=0) == rows(M=5) == rows(K=8193, ws=8208) == rows(ws=16) == rows(ys=19) == rows(xs=-1) == -12
    assert rows(x=258) == rows(w=260) == rows(ws=40) == -6
