"""A training step that is warmed up on a side stream and captured on another while the warm-up's loss is still held: the leaves' gradients are then summed on the
side stream, which the capture takes in and joins again."""
import pytest
import torch

gpu = pytest.mark.gpu


def data(seed, M=700, V=3000, K=64, dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    table = (torch.randn((V, K), generator=gen, device="cuda") * 0.1).to(dtype)
    return table, torch.randint(V, (M,), generator=gen, device="cuda"), torch.randint(-1, V, (M,), generator=gen, device="cuda")


def loss_of(table, tokens, targets):
    import rapid_sampling_amd as sample
    return sample.linear_cross_entropy(sample.embedding(tokens, table, 2.0), table, targets, 0.9).loss.sum()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("how", ["backward", "grad"])
def test_the_warm_up_is_still_held(how, dtype):
    from tests.test_operator_workspaces import fresh_stream
    print("captured", how, dtype, flush=True)
    table, tokens, targets = data(1, dtype=dtype)
    leaf = table.clone().requires_grad_()
    warm, side = fresh_stream(), fresh_stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        for _ in range(2):
            leaf.grad = None
            loss = loss_of(leaf, tokens, targets)
            loss.backward()
    torch.cuda.current_stream().wait_stream(warm)
    leaf.grad = None
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = loss_of(leaf, tokens, targets)
        if how == "backward":
            held.backward()
            grad = leaf.grad
        else:
            grad, = torch.autograd.grad(held, leaf)
    assert loss.grad_fn is not None                                      # (the warm-up's graph)
    for seed in range(4):
        fresh, new_tokens, new_targets = data(10 + seed, dtype=dtype)
        with torch.no_grad():
            leaf.copy_(fresh)
        tokens.copy_(new_tokens)
        targets.copy_(new_targets)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = fresh.clone().requires_grad_()
        want = loss_of(eager, new_tokens, new_targets)
        want.backward()
        assert torch.equal(held, want) and torch.equal(grad, eager.grad), seed


@gpu
def test_one_operator_alone():
    """Embedding's table, and x and the weight of the loss, each held by a graph of the side stream."""
    import rapid_sampling_amd as sample
    from tests.test_operator_workspaces import fresh_stream
    table, tokens, targets = data(2)
    x = (torch.randn((700, 64), generator=torch.Generator().manual_seed(1)) * 0.5).bfloat16().cuda()
    g = torch.ones((700, 64), dtype=torch.bfloat16, device="cuda")
    for call, leaves in ((lambda a, b: (sample.embedding(tokens, b) * g).sum(), 1), (lambda a, b: sample.linear_cross_entropy(a, b, targets).loss.sum(), 2)):
        a, b = x.clone().requires_grad_(), table.clone().requires_grad_()
        warm, side = fresh_stream(), fresh_stream()
        warm.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(warm):
            kept = call(a, b)
            kept.backward()
        torch.cuda.current_stream().wait_stream(warm)
        want = b.grad, a.grad
        a.grad = b.grad = None
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call(a, b).backward()
        for _ in range(3):
            b.grad.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(b.grad, want[0]) and (leaves == 1 or torch.equal(a.grad, want[1]))
        del kept
