"""The sums of token_logprobs where they are exact, so that one term left out or taken twice shows.

With temperature log2(e) a logit of -n weighs 2^-n.  A row of equal logits has S = V and entropy ln V; one of a zeros and b logits of -8 has
256 S = 256 a + b, a whole number below 2^24, and -sum e z / S = 8 ln 2 b / (256 S).  What is left are the logarithm, a quotient and three
roundings: 4 units in the last place of results of up to 16, 2^-18 of the smaller ones; a term of 131072 left out is 2 ^ -17."""
import math

import pytest
import torch

TEMPERATURE = 1.4426950408889634
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LIMIT = 2.0 ** -18

pytestmark = pytest.mark.gpu


def look(x, low, top):
    """x: rows of 0 and -8, `low` of the latter in each."""
    import rapid_sampling_amd as sample
    rows, V = x.shape
    t = (torch.arange(rows, device="cuda") * 7919) % V
    out = sample.token_logprobs(x, t, TEMPERATURE, top=top)
    low = low.double().cpu()
    S = (V - low) + low / 256
    entropy = torch.log(S) + 8 * math.log(2) * (low / 256) / S
    z = x.gather(1, t[:, None])[:, 0].double().cpu() * math.log(2)
    assert (out.logprobs.double().cpu() - (z - torch.log(S))).abs().max() < LIMIT
    assert (out.entropy.double().cpu() - entropy).abs().max() < LIMIT
    z = x.gather(1, out.top_tokens.long()).double().cpu() * math.log(2)
    assert ((out.top_logprobs.double().cpu() - (z - torch.log(S)[:, None])).abs() < LIMIT).all()
    index = torch.arange(V, device="cuda")
    first = [(torch.nonzero(row == 0)[:, 0].tolist() + torch.nonzero(row < 0)[:, 0].tolist())[:top] for row in x[:5]]
    assert out.top_tokens[:5].tolist() == first
    x_t = x.gather(1, t[:, None])
    for part in range(0, rows, 256):
        xs, ts = x[part:part + 256], t[part:part + 256, None]
        rank = 1 + ((xs > x_t[part:part + 256]) | ((xs == x_t[part:part + 256]) & (index < ts))).sum(-1)
        assert torch.equal(rank.int(), out.rank[part:part + 256])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,V", [(1, 65536), (3, 131072), (1, 50257), (30, 20001), (200, 5003), (700, 9001), (2100, 600), (2100, 16000), (2500, 77)])
def test_sums_that_are_exact(rows, V, dtype):
    print("exact", rows, V, dtype, flush=True)
    gen = torch.Generator(device="cuda").manual_seed(rows + V)
    for top in (0, 1, 20):
        look(torch.zeros((rows, V), device="cuda", dtype=DTYPES[dtype]), torch.zeros(rows), top)
        if V > 65535:
            continue
        x = torch.where(torch.rand((rows, V), generator=gen, device="cuda") < 0.5, -8.0, 0.0).to(DTYPES[dtype])
        look(x, (x < 0).sum(-1), top)
