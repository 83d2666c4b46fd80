"""The workspaces of token_logprobs and linear_fp8: reserved before a capture whatever the vocabulary, left out where they are not wanted, and
nothing beside them and the outputs."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu


def fresh_stream():
    """A stream that no call has used yet (torch's own come from a pool)."""
    h = C.c_void_p()
    assert C.CDLL("libamdhip64.so").hipStreamCreate(C.byref(h)) == 0
    return torch.cuda.ExternalStream(h.value)


def inputs(V, K=256, B=3, seed=1):
    import rapid_sampling_amd as sample
    gen = torch.Generator(device="cuda").manual_seed(seed)
    w, s = sample.quantize_fp8(torch.randn((V, K), generator=gen, device="cuda"), block_rows=128)
    hidden = torch.randn((B, K), generator=gen, device="cuda", dtype=torch.bfloat16)
    return hidden, w, s, torch.randint(0, V, (B,), generator=gen, device="cuda")


@pytest.mark.parametrize("V", [50257, 1001, 4096])
def test_reserved_for_any_vocabulary(V):
    import rapid_sampling_amd as sample
    hidden, w, s, t = inputs(V)

    def step(h):
        logits = sample.linear_fp8(h, w, s)
        return (logits,) + tuple(sample.token_logprobs(logits, t, 0.9, top=5))
    step(hidden)                                            # (the kernels are loaded)
    torch.cuda.synchronize()
    side = fresh_stream()
    held_in = hidden.clone()
    with torch.cuda.stream(side):
        sample.reserve_workspace(3, V)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step(held_in)
    for seed in range(3):
        held_in.copy_(inputs(V, seed=10 + seed)[0])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step(held_in))), seed


def test_left_out_where_they_are_not_wanted():
    import rapid_sampling_amd as sample
    torch.cuda.synchronize()

    def taken(**kw):
        with torch.cuda.stream(fresh_stream()):
            before = torch.cuda.memory_allocated()
            sample.reserve_workspace(2, 4096, **kw)
            return torch.cuda.memory_allocated() - before
    both, alone = taken(), taken(operators=False)
    assert 12 << 20 < both - alone < 13 << 20
    hidden, w, s, t = inputs(4096)
    logits = sample.linear_fp8(hidden, w, s)
    side = fresh_stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        sample.reserve_workspace(3, 4096, operators=False)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            with pytest.raises(RuntimeError, match="reserve_workspace"):
                sample.token_logprobs(logits, t)
            hidden.add_(0)
    torch.cuda.synchronize()


def test_refused_sizes():
    import rapid_sampling_amd as sample
    for B, V in ((1, 0), (1, -3), (1, 1048577), (0, 8)):
        with pytest.raises(ValueError):
            sample.reserve_workspace(B, V)


def test_calls_allocate_their_outputs_and_nothing_that_stays():
    """Device memory in use before and after calls through the C ABI, which allocates nothing at all, and through the module, whose outputs are
    all that is there while they are kept."""
    import rapid_sampling_amd as sample
    from tests import capi
    L = capi.lib()
    hidden, w, s, t = inputs(4096, B=40)
    logits = sample.linear_fp8(hidden, w, s)
    p, i32, i64, size = C.c_void_p, C.c_int32, C.c_int64, C.c_size_t
    L.rs_logprobs_workspace_bytes.restype = L.rs_linear_workspace_bytes.restype = size
    L.rs_token_logprobs.argtypes = [p, i32, i64, i64, p, i32, i64, i64, i32, i32, i32, C.c_double, i32] + [p] * 6 + [p, size, p]
    L.rs_linear_blocks.argtypes = [p, i64, p, p, i64, p, i32, i32, i32, p, i32, i64, p, size, p]
    L.rs_quantize_blocks.argtypes = [p, i32, i64, i32, i32, i32, p, i64, p, p]
    L.rs_workspace_init.argtypes = [p, size, p]
    spaces = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in (L.rs_logprobs_workspace_bytes(), L.rs_linear_workspace_bytes())]
    st = torch.cuda.current_stream().cuda_stream
    for ws in spaces:
        assert L.rs_workspace_init(ws.data_ptr(), ws.numel(), st) == 0
    q, scale = sample.quantize_fp8(hidden)
    y, outs = torch.empty_like(logits), [torch.empty(40, dtype=torch.int32, device="cuda") for _ in range(3)]
    top = [torch.empty((40, 5), dtype=torch.int32, device="cuda") for _ in range(2)]

    def calls():
        assert L.rs_quantize_blocks(hidden.data_ptr(), 1, 256, 1, 40, 256, q.data_ptr(), 256, scale.data_ptr(), st) == 0
        assert L.rs_linear_blocks(q.data_ptr(), 256, scale.data_ptr(), w.data_ptr(), 256, s.data_ptr(), 40, 4096, 256, y.data_ptr(), 0, 4096,
                                  spaces[1].data_ptr(), spaces[1].numel(), st) == 0
        assert L.rs_token_logprobs(y.data_ptr(), 0, 4096, 0, t.data_ptr(), 1, 1, 0, 40, 1, 4096, 0.9, 5, *[o.data_ptr() for o in outs + top], None,
                                   spaces[0].data_ptr(), spaces[0].numel(), st) == 0
    calls()
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(3):
        calls()
    torch.cuda.synchronize()
    assert torch.cuda.mem_get_info()[0] == free
    want = sample.token_logprobs(logits, t, 0.9, top=5)
    assert torch.equal(y, logits) and torch.equal(outs[2], want.rank) and torch.equal(top[1], want.top_tokens)
    assert torch.equal(outs[0].view(torch.float32), want.logprobs)
    before = torch.cuda.memory_allocated()
    for _ in range(3):
        sample.token_logprobs(sample.linear_fp8(hidden, w, s), t, 0.9, top=5)
    assert torch.cuda.memory_allocated() == before
