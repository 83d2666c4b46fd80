"""What linear_fp8's sums hold, in every kernel that it chooses from and for every type of output.

Whole numbers whose sums fit 24 bits come out exactly, in whatever order they are added, and are rounded once: large products that
cancel beside small ones are such numbers.

For random columns the root of the mean square says more than a bound on each: each of n = 128 + 2 blocks roundings is off by eps = 2^-24 of
a partial sum at most (2 eps where a sum is cut off in the place of rounded), with chance signs, and partial sums are no larger in the mean than
the result: 4 eps sqrt(n) of the results' own root mean square, twice what is expected, beside half a unit of the output's type.  Of 4096
columns one left out is 1.6e-2 of it, of 300 5.8e-2."""
import math

import pytest
import torch

EPS = 2.0 ** -24
F8 = torch.float8_e4m3fn
OUT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
# few rows; tiles of 128 x 64, their columns shared out or not; tiles of 128 x 128, with whole and other last blocks, rows and columns
SHAPES = [(3, 300, 1000), (12, 4096, 700), (40, 4096, 515), (40, 200, 3000), (100, 1000, 1037), (200, 384, 640), (77, 300, 33001), (77, 1999, 33001),
          (300, 130, 16400), (300, 1000, 16400), (500, 384, 32800), (256, 512, 65500), (256, 1024, 32768)]

pytestmark = pytest.mark.gpu


def quantized(R, K, seed, rows):
    """Values in 8 bits and their scales, made without the framework."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((R, K), generator=gen, device="cuda") * torch.exp(torch.randn((K,), generator=gen, device="cuda"))
    q = torch.zeros((R, K + -K % 16), dtype=torch.uint8, device="cuda").view(F8)
    q[:, :K] = (x * 8).clamp(-448, 448).to(F8)
    scale = torch.rand((-(-R // rows), -(-K // 128)), generator=gen, device="cuda") + 0.5
    return q[:, :K], scale


def wide(q, scale, rows):
    at = torch.arange(q.shape[0], device="cuda") // rows
    columns = torch.arange(q.shape[1], device="cuda") // 128
    return q.double() * scale.double()[at][:, columns]


@pytest.mark.parametrize("out", list(OUT))
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_sums_of_random_columns(M, K, N, out):
    import rapid_sampling_amd as sample
    print("sums", M, K, N, out, flush=True)
    (x, sx), (w, sw) = quantized(M, K, M + K, 1), quantized(N, K, N + K, 128)
    y = sample.linear_fp8(x, w, sw, x_scale=sx, out_dtype=OUT[out])
    assert y.dtype == OUT[out] and y.shape == (M, N)
    # the first columns, some in the middle, the last ones
    some = torch.cat([torch.arange(0, min(N, 300)), torch.arange(N // 2, min(N, N // 2 + 300)), torch.arange(max(0, N - 300), N)]).unique().cuda()
    want = wide(x, sx, 1) @ wide(w.view(torch.uint8)[some].view(F8), sw[some // 128], 1).T
    got = y[:, some].double()
    # beyond the type's range (float16's sums reach it here) there is nothing but an infinity of the sum's sign
    over = want.abs() > torch.finfo(OUT[out]).max
    assert torch.equal(got.isinf() | over, over) and torch.equal(got[got.isinf()].sign(), want[got.isinf()].sign())
    off = torch.where(got.isinf(), 0.0, got - want)
    size = want.square().mean().sqrt()
    bound = (4 * EPS * math.sqrt(128 + 2 * sx.shape[1]) + UNIT[out]) * size
    for rows in (off[:16], off[-16:], off):                             # (a tile's first and last rows by themselves)
        assert rows.square().mean().sqrt() <= bound, (rows.square().mean().sqrt() / size).item()
    for columns in (off[:, :16], off[:, -16:]):
        assert columns.square().mean().sqrt() <= 4 * bound, (columns.square().mean().sqrt() / size).item()


@pytest.mark.parametrize("out", list(OUT))
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_large_products_that_cancel(M, K, N, out):
    """256 * 256 - 256 * 256 beside products of 0 to 16, in every eight columns: exact, whichever is added first."""
    import rapid_sampling_amd as sample
    print("cancel", M, K, N, out, flush=True)
    gen = torch.Generator(device="cuda").manual_seed(M + K + N)
    x = torch.randint(0, 5, (M, K), generator=gen, device="cuda").float()
    w = torch.randint(-4, 5, (N, K), generator=gen, device="cuda").float()
    for at in range(0, K - 7, 8):
        first, second = torch.randperm(8, generator=torch.Generator().manual_seed(at))[:2].tolist()
        x[:, at + first], x[:, at + second] = 256.0, 256.0
        w[:, at + first], w[:, at + second] = 256.0, -256.0
    want = (x.double() @ w.double().T).to(OUT[out])
    held_x = torch.zeros((M, K + -K % 16), dtype=torch.uint8, device="cuda").view(F8)
    held_w = torch.zeros((N, K + -K % 16), dtype=torch.uint8, device="cuda").view(F8)
    held_x[:, :K], held_w[:, :K] = x.to(F8), w.to(F8)
    blocks = -(-K // 128)
    one_x, one_w = torch.ones((M, blocks), device="cuda"), torch.ones((-(-N // 128), blocks), device="cuda")
    y = sample.linear_fp8(held_x[:, :K], held_w[:, :K], one_w, x_scale=one_x, out_dtype=OUT[out])
    assert torch.equal(y, want), (y.double() - want.double()).abs().max().item()
