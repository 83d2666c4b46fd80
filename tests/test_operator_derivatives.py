"""Derivatives that the operators next to the sampler do not have are refused where they are asked for, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

F8 = torch.float8_e4m3fn


def inputs(device):
    gen = torch.Generator().manual_seed(1)
    x, w, s = torch.randn((2, 32), generator=gen), torch.zeros((16, 32), dtype=torch.uint8).view(F8), torch.ones((1, 1))
    return x.to(device), w.to(device), s.to(device), torch.zeros(2, dtype=torch.long, device=device)


def tangents(device):
    import rapid_sampling_amd as sample
    x, w, s, t = inputs(device)
    with fwd.dual_level():
        dual, dual_scale = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(s, torch.ones_like(s))
        for call in (lambda: sample.token_logprobs(dual, t), lambda: sample.token_logprobs(dual.detach().requires_grad_() * dual, t),
                     lambda: sample.linear_fp8(dual, w, s), lambda: sample.linear_fp8(x, w, dual_scale), lambda: sample.quantize_fp8(dual)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):         # (which does not turn these off)
                call()
        return dual, fwd.unpack_dual(dual).primal


def test_forward_mode_is_refused():
    tangents("cpu")


@pytest.mark.gpu
def test_forward_mode_is_refused_on_the_gpu():
    import rapid_sampling_amd as sample
    x, w, s, t = inputs("cuda")
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        primal = fwd.unpack_dual(dual).primal
        assert torch.equal(sample.token_logprobs(primal, t).logprobs, sample.token_logprobs(x, t).logprobs)
    tangents("cuda")
    assert torch.equal(sample.token_logprobs(dual, t).logprobs, sample.token_logprobs(x, t).logprobs)          # its level is over


@pytest.mark.gpu
@pytest.mark.parametrize("again", [False, True])
def test_forward_mode_over_the_gradient_is_refused(again):
    """A tangent that comes in with the outputs' gradients, by a factor of the loss."""
    import rapid_sampling_amd as sample
    x, _, _, t = inputs("cuda")
    x.requires_grad_()
    out = sample.token_logprobs(x, t, top=3)
    with fwd.dual_level():
        for value in (out.logprobs, out.entropy, out.top_logprobs):
            factor = fwd.make_dual(torch.ones_like(value), torch.ones_like(value))
            with pytest.raises((RuntimeError, ValueError), match="forward-mode"):
                torch.autograd.grad((value * factor).sum(), x, retain_graph=True, create_graph=again)
    grad, = torch.autograd.grad(out.entropy.sum(), x)
    assert grad.abs().sum() > 0


def test_weights_that_ask_for_a_gradient_are_refused():
    """A Parameter of any floating type asks for one unless it is told not to."""
    import rapid_sampling_amd as sample
    x, w, s, _ = inputs("cpu")
    learnt, scale = torch.nn.Parameter(w), torch.nn.Parameter(s)
    assert learnt.requires_grad
    for args in ((x, learnt, s), (x, w, scale), (x.clone().requires_grad_(), w, s)):
        with pytest.raises(ValueError, match="no gradient"):
            sample.linear_fp8(*args)
        with torch.no_grad(), pytest.raises(ValueError, match="GPU"):                       # (asked for none: the next check)
            sample.linear_fp8(*args)
    with pytest.raises(ValueError, match="GPU"):
        sample.linear_fp8(x, torch.nn.Parameter(w, requires_grad=False), s)


@pytest.mark.gpu
def test_a_frozen_parameter_is_a_weight():
    import rapid_sampling_amd as sample
    x, w, s, _ = inputs("cuda")
    w = torch.randn((16, 32), device="cuda").to(F8)
    y = sample.linear_fp8(x, w, s)
    assert torch.equal(sample.linear_fp8(x, torch.nn.Parameter(w, requires_grad=False), s), y)
    with torch.no_grad():
        assert torch.equal(sample.linear_fp8(x, torch.nn.Parameter(w), s), y)
    with pytest.raises(ValueError, match="no gradient"):
        sample.linear_fp8(x, torch.nn.Parameter(w), s)
