#!/usr/bin/env python3
"""A decode loop from hidden states to answers, and a step of policy gradient on what it sampled.

An 8-bit head makes the logits (linear_fp8), the sampler draws a token for each row, and token_logprobs says how likely it
was, which rank it had and what the alternatives were.  Then the same tokens are scored again, under autograd, and the
gradient of a policy-gradient loss with an entropy bonus goes back to the logits.

    python examples/head_and_logprobs.py
"""
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

import torch

import rapid_sampling_amd as sample


def main(batch=4, hidden_size=1024, vocab=32768, steps=3, temperature=0.8, top_k=50, top_p=0.95, alternatives=5, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    # once, as the model is loaded: the head's weight in 8 bits, with a scale for each block of 128 x 128
    weight = torch.randn((vocab, hidden_size), generator=gen, device="cuda") * 0.05
    head, head_scale = sample.quantize_fp8(weight, block_rows=128)
    states = sample.setup_rand(seed, batch)

    hidden, tokens, answers = [], [], []
    for step in range(steps):
        h = torch.randn((batch, hidden_size), generator=gen, device="cuda").bfloat16()     # a model's last hidden states
        logits = sample.linear_fp8(h, head, head_scale)
        token = sample.batch_sampling_temperature_topk_topp(logits, states, temperature, top_k, top_p)
        answer = sample.token_logprobs(logits, token, temperature, top=alternatives)
        print("step %d:" % step, [(t, "%.2f" % lp, "rank %d" % r) for t, lp, r in
                                  zip(token.tolist(), answer.logprobs.tolist(), answer.rank.tolist())])
        hidden.append(h)
        tokens.append(token)
        answers.append(answer)

    # the rollout once more, all positions at a time, with a gradient
    hidden, tokens = torch.stack(hidden, dim=1), torch.stack(tokens, dim=1)
    logits = sample.linear_fp8(hidden, head, head_scale, out_dtype=torch.bfloat16).requires_grad_()
    scored = sample.token_logprobs(logits, tokens, temperature)
    advantage = torch.randn(tokens.shape, generator=gen, device="cuda")
    loss = -(advantage * scored.logprobs).mean() - 0.01 * scored.entropy.mean()
    loss.backward()
    print("loss %.4f, gradient" % loss.item(), tuple(logits.grad.shape), "entropy per position %.3f" % scored.entropy.mean().item())
    return answers, scored, logits.grad


if __name__ == "__main__":
    main()
