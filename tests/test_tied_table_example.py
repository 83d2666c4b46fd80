"""The example of a tied table runs, and its gradients are those of its formula in 64 bits and of differences."""
import runpy

import pytest
import torch

from tests.conftest import ROOT

gpu = pytest.mark.gpu


def example():
    return runpy.run_path(ROOT + "/examples/tied_table.py")


def formula(table, mix, tokens, targets, auxiliary=1e-2):
    """The example's loss in float64, by plain operations."""
    rows = table[tokens.clamp(min=0)] * (tokens >= 0)[..., None]
    logits = torch.tanh(rows * table.shape[1] ** 0.5 @ mix) @ table.T
    lse = torch.logsumexp(logits, -1)
    there = targets >= 0
    picked = torch.gather(logits, -1, targets.clamp(min=0)[..., None])[..., 0]
    return (there * (lse - picked + auxiliary * lse.square())).sum() / there.sum()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_example(dtype):
    """Rounding units on the way, each of the type's u: the table's and the layer's are the inputs' own.  The loss and each gradient pass fewer
    than 16 roundings to the type one after the other (looked up row, product, tanh, its two derivatives, G, dx, the two parts of the table's
    gradient and their sum), each of at most u of its result; the tanh halves what goes in or leaves it as it is, and the logits' errors
    (below 4 u of logits below 8) come into G as a factor of at most 1 + 32 u.  Together below 64 u in the norm of a gradient, and float32's sums
    of up to 5000 terms, in parts of 32 at most one after the other, stay below that."""
    run = example()["main"]
    loss, table, mix, tokens, targets, answers = run(dtype=dtype)
    u = torch.finfo(dtype).eps / 2
    t, m = table.detach().double().cpu().requires_grad_(), mix.detach().double().cpu().requires_grad_()
    want = formula(t, m, tokens.cpu(), targets.cpu())
    want.backward()
    assert abs(loss.item() - want.item()) <= 64 * u * want.item()
    for got, ref in ((table.grad, t.grad), (mix.grad, m.grad)):
        assert (got.double().cpu() - ref).norm() <= 64 * u * ref.norm()
    assert all(torch.isfinite(a.logprobs).all() and (a.rank <= 50).all() for a in answers)


@gpu
def test_differences():
    """Along a direction d the loss in float32 changes by what the gradients say: over 2 h the loss (about 9, off by 64 units 2^-24 of it at most) differs
    from the line by its third derivative, h^2 / 6 of it."""
    ns = example()
    loss, table, mix, tokens, targets, _ = ns["main"](dtype=torch.float32)
    gen = torch.Generator(device="cuda").manual_seed(5)
    dt, dm = torch.randn(table.shape, generator=gen, device="cuda") * 0.02, torch.randn(mix.shape, generator=gen, device="cuda") * 0.02
    dt, dm = dt + table.grad, dm + mix.grad                      # (a direction along which the loss does change)
    slope = ((table.grad * dt).sum() + (mix.grad * dm).sum()).item()
    h = 0.05
    with torch.no_grad():
        ends = [ns["forward"](table + s * h * dt, mix + s * h * dm, tokens, targets)[0].item() for s in (1, -1)]
        wide = [ns["forward"](table + 2 * s * h * dt, mix + 2 * s * h * dm, tokens, targets)[0].item() for s in (1, -1)]
    # two distances cancel the third derivative: (8 (f(h) - f(-h)) - (f(2h) - f(-2h))) / 12 h, off by the fifth; 18 / 12 h of the loss's own error
    got = (8 * (ends[0] - ends[1]) - (wide[0] - wide[1])) / (12 * h)
    assert abs(got - slope) <= 18 / (12 * h) * 64 * 2 ** -24 * loss.item() + 1e-3 * abs(slope)


@gpu
def test_a_captured_step_beside_an_eager_graph():
    """A training step is captured, and replayed, with both gradients of the table; while an eager graph of the table from another stream lives the
    capture is refused, and goes through once that is gone."""
    import rapid_sampling_amd as sample
    from tests.test_operator_workspaces import fresh_stream
    gen = torch.Generator(device="cuda").manual_seed(3)
    table = (torch.randn((3000, 64), generator=gen, device="cuda") * 0.1).requires_grad_()
    tokens = torch.randint(3000, (700,), generator=gen, device="cuda")
    eager = sample.embedding(tokens, table)
    side = fresh_stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            spare = torch.zeros(4, device="cuda")
            for call in (lambda: sample.embedding(tokens, table), lambda: sample.linear_cross_entropy(table[:700].detach(), table, tokens)):
                with pytest.raises(RuntimeError, match="another stream lives"):
                    call()
            spare.add_(1)
        del eager
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            loss = sample.linear_cross_entropy(sample.embedding(tokens, table, 2.0), table, tokens).loss.sum()
            loss.backward()
    held = table.grad
    for seed in range(4):
        tokens.copy_(torch.randint(3000, (700,), generator=gen, device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        fresh = table.detach().clone().requires_grad_()
        sample.linear_cross_entropy(sample.embedding(tokens, fresh, 2.0), fresh, tokens).loss.sum().backward()
        assert torch.equal(held, fresh.grad), seed
