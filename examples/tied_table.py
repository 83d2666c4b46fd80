#!/usr/bin/env python3
"""One table at both ends: a training step, and then a decode loop that is served from the table in 8-bit integers.

The tokens' rows (embedding) go through a small layer, and the loss is taken against the same table (linear_cross_entropy), so its
gradient has two parts: from the rows that were looked up and from the head.  An auxiliary loss keeps the logsumexp near 0.
For serving the table is rounded once (quantize_int8); each step looks the last tokens up in it, makes logits with it
(linear_int8), draws the next tokens and says how likely they were (token_logprobs).

    python examples/tied_table.py
"""
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

import torch

import rapid_sampling_amd as sample


def forward(table, mix, tokens, targets, auxiliary=1e-2):
    """Mean loss over the targets that are there (not negative), with auxiliary * logsumexp^2."""
    hidden = torch.tanh(sample.embedding(tokens, table, table.shape[1] ** 0.5) @ mix)
    out = sample.linear_cross_entropy(hidden, table, targets)
    there = targets >= 0
    loss = (out.loss + auxiliary * there * out.logsumexp.square()).sum() / there.sum()
    return loss, hidden


def main(batch=4, length=40, hidden_size=256, vocab=5000, steps=3, temperature=0.8, top_k=50, top_p=0.95, seed=0, dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    table = (torch.randn((vocab, hidden_size), generator=gen, device="cuda") * hidden_size ** -0.5).to(dtype).requires_grad_()
    mix = (torch.randn((hidden_size, hidden_size), generator=gen, device="cuda") * hidden_size ** -0.5).to(dtype).requires_grad_()
    text = torch.randint(vocab, (batch, length + 1), generator=gen, device="cuda")
    text[:, -3:] = -1                                            # padding: no row, no loss
    tokens, targets = text[:, :-1], text[:, 1:]

    loss, _ = forward(table, mix, tokens, targets)
    loss.backward()
    print("loss %.4f, gradients" % loss.item(), tuple(table.grad.shape), tuple(mix.grad.shape))

    answers = []
    with torch.no_grad():
        q, scale = sample.quantize_int8(table)
        states = sample.setup_rand(seed, batch)
        token = text[:, 0]
        for step in range(steps):
            hidden = torch.tanh(sample.embedding(token, q, hidden_size ** 0.5, weight_scale=scale, out_dtype=dtype) @ mix)
            logits = sample.linear_int8(hidden, q, scale)
            token = sample.batch_sampling_temperature_topk_topp(logits, states, temperature, top_k, top_p)
            answers.append(sample.token_logprobs(logits, token, temperature))
            print("step %d:" % step, token.tolist(), ["%.2f" % lp for lp in answers[-1].logprobs.tolist()])
    return loss.detach(), table, mix, tokens, targets, answers


if __name__ == "__main__":
    main()
