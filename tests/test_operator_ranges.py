"""Calls of the operators next to the sampler with more rows than one launch takes: their last rows, and those where one launch ends and the
next begins, against the same rows by themselves.  Everything else about them is small."""
import ctypes as C

import pytest
import torch

F8 = torch.float8_e4m3fn
gpu = pytest.mark.gpu


def places(rows, *ends):
    """The first rows, the last ones, and those about the ends of launches."""
    return torch.cat([torch.arange(3)] + [torch.arange(e - 2, e + 2) for e in ends] + [torch.arange(rows - 3, rows)]).cuda()


def near(a, b):
    return torch.allclose(a, b, rtol=0, atol=2.0 ** -24 * 400 * 10) if a.is_floating_point() else torch.equal(a, b)


@gpu
@pytest.mark.parametrize("rows,V,top,end", [((1 << 24) + 3, 34, 33, (1 << 24) - 1), ((1 << 26) + 3, 9, 2, (1 << 26) - 1)])
def test_rows_of_logits(rows, V, top, end):
    import rapid_sampling_amd as sample
    print("rows", rows, V, top, flush=True)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((rows, V), generator=gen, device="cuda", dtype=torch.bfloat16)
    t = torch.randint(0, V, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    some = places(rows, end)
    part = x[some].clone().requires_grad_()
    want = sample.token_logprobs(part, t[some], 0.9, top=top)
    got = sample.token_logprobs(x, t, 0.9, top=top)
    assert all(near(a[some], b.detach()) for a, b in zip(got, want))
    assert (got.rank >= 1).all() and (got.rank <= V).all() and (got.top_tokens >= 0).all() and (got.top_tokens < V).all()
    del got
    if top > 32:
        return
    want.logprobs.sum().backward()
    x.requires_grad_()
    sample.token_logprobs(x, t, 0.9).logprobs.sum().backward()
    assert near(x.grad[some], part.grad) and not x.grad.isnan().any()


@gpu
@pytest.mark.parametrize("R,K,rows,end", [((1 << 28) + 5, 1, 1, 16 * ((1 << 24) - 1)), ((1 << 27) + 40, 129, 1, 8 * ((1 << 24) - 1)),
                                          ((1 << 31) - 1, 1, 128, 128 * ((1 << 24) - 1))])
def test_blocks_of_values(R, K, rows, end):
    import rapid_sampling_amd as sample
    print("blocks", R, K, rows, flush=True)
    gen = torch.Generator(device="cuda").manual_seed(2)
    if K == 1:
        x = torch.randn((R, K), generator=gen, device="cuda", dtype=torch.bfloat16)
    else:                                                           # rows that overlap: K values from each one on
        x = torch.randn((R + K,), generator=gen, device="cuda", dtype=torch.bfloat16).as_strided((R, K), (1, 1))
    q, scale = sample.quantize_fp8(x, block_rows=rows)
    for first, last in ((0, 256), (end - 256, end + 128), ((R - 200) // 128 * 128, R)):
        want, want_scale = sample.quantize_fp8(x[first:last].clone() if rows == 128 else x[first:last], block_rows=rows)
        assert torch.equal(q[first:last].view(torch.uint8), want.view(torch.uint8))
        assert torch.equal(scale[first // rows: -(-last // rows)], want_scale)


@gpu
def test_rows_of_a_product_with_a_weight_whose_rows_lie_far_apart():
    """Whole numbers from -8 to 8, which are 56 / 448 of the largest and more once rounded: their sums are exact, by any kernel."""
    import rapid_sampling_amd as sample
    M, K, N = (1 << 20) + 5, 16, 2
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(-8, 9, (M, K), generator=gen, device="cuda").bfloat16()
    store = torch.zeros((N, 1 << 24), dtype=torch.uint8, device="cuda")
    w, w_scale = sample.quantize_fp8(torch.randint(-8, 9, (N, K), generator=gen, device="cuda").float(), block_rows=128)
    store[:, :K] = w.view(torch.uint8)
    for out in (torch.float32, torch.bfloat16):
        y = sample.linear_fp8(x, store.view(F8)[:, :K], w_scale, out_dtype=out)
        assert torch.equal(y, sample.linear_fp8(x, w, w_scale, out_dtype=out))


def test_products_of_more_tiles_than_a_launch_holds_are_refused():
    from tests import capi
    L = capi.lib()
    p, i32, i64 = C.c_void_p, C.c_int32, C.c_int64
    L.rs_linear_workspace_bytes.restype = C.c_size_t
    n = L.rs_linear_workspace_bytes()
    L.rs_linear_blocks.argtypes = [p, i64, p, p, i64, p, i32, i32, i32, p, i32, i64, p, C.c_size_t, p]

    def linear(M, N):
        return L.rs_linear_blocks(256, 32, 256, 256, 32, 256, M, N, 20, 256, 0, N, 256, n, None)
    assert linear(1 << 24, 1 << 14) == linear(1 << 24, 1 << 24) == linear(128 * 4096, 128 * 4096) == -12
    assert linear(1 << 25, 1) == linear(1, 1 << 25) == -12
