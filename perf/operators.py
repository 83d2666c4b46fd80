"""The operators next to the sampler whose time is followed: what is answered and learnt about sampled tokens
(`token_logprobs` and its gradient) and the 8-bit head that makes the logits (`linear_fp8`).

A case is a dict of plain values.  "op" is one of

  "logprobs"  log probabilities, entropies, ranks and `top` alternatives of given tokens, as a serving or a
              scoring program asks for them
  "gradient"  the same call under autograd and the gradient of its logits, as a training step makes it
  "linear"    y = x W^T with W in 8 bits and a scale for each block of 128 x 128; x in 16 or 32 bits, quantised within the
              call in blocks of 1 x 128, or (x_dtype "float8") in 8 bits already

and the rest are sizes:

  B, T, V      shape of the logits: (B, V) where T is 0, else (B, T, V) -- the first T of T + 1 positions, since the last
               one predicts nothing that is given
  dtype        of the logits; masked: share of the vocabulary (its end) that is -inf, as a padded vocabulary is
  M, K, N      rows of x, hidden size, rows of W; x_dtype, out_dtype
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK, FP8_MAX, SCALE_MIN = 128, 448.0, 2.0 ** -126


def _rows(op, B, T, V, dtype, top, temperature=1.0, masked=0.0):
    return {"op": op, "B": B, "T": T, "V": V, "dtype": dtype, "top": top, "temperature": temperature, "masked": masked}


def _linear(M, K, N, x_dtype="bfloat16", out_dtype="float32"):
    return {"op": "linear", "M": M, "K": K, "N": N, "x_dtype": x_dtype, "out_dtype": out_dtype}


def listed():
    cases = [
        # one user's decode loop that answers with the token's log probability and five alternatives
        ("logprobs_one_row", _rows("logprobs", 1, 0, 65536, "float32", 5)),
        # a serving batch with the most alternatives that services offer
        ("logprobs_batch", _rows("logprobs", 64, 0, 152064, "bfloat16", 20, temperature=0.8)),
        # scoring a few texts: an odd vocabulary, so that rows begin at any address, padded with masked tokens
        ("logprobs_ragged", _rows("logprobs", 7, 129, 50257, "float16", 1, masked=0.01)),
        # scoring a batch of prompts
        ("logprobs_prompts", _rows("logprobs", 16, 512, 131072, "bfloat16", 20)),
        # a small policy-gradient step in float32
        ("gradient_small", _rows("gradient", 48, 0, 32768, "float32", 0)),
        # distillation on the 64 likeliest tokens, odd sizes
        ("gradient_ragged", _rows("gradient", 5, 77, 50257, "float16", 64, temperature=1.5, masked=0.01)),
        # a training step on rollouts: log probabilities and an entropy bonus
        ("gradient_rollouts", _rows("gradient", 8, 1024, 131072, "bfloat16", 0, temperature=0.9)),
        # the head of one user's decode loop
        ("linear_one_row", _linear(1, 4096, 65536)),
        # the head of a serving batch
        ("linear_batch", _linear(32, 4096, 131072)),
        # odd sizes: a hidden size that is no whole number of blocks, an odd vocabulary
        ("linear_ragged", _linear(77, 2000, 50257, x_dtype="float16", out_dtype="bfloat16")),
        # the head over a prompt, for scoring
        ("linear_prompts", _linear(4096, 4096, 131072, out_dtype="bfloat16")),
        # a square projection, activations quantised by the layer before
        ("linear_square", _linear(8192, 8192, 8192, x_dtype="float8", out_dtype="bfloat16")),
    ]
    return [dict(c, name=name) for name, c in cases]


def _log_uniform(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "gradient", "linear", "linear"])
    if op == "linear":
        K = _log_uniform(rng, 256, 8192)
        N = _log_uniform(rng, 512, 131072)
        M = _log_uniform(rng, 1, min(8192, max(1, (1 << 40) // (K * N))))
        return _linear(M, K, N, x_dtype=rng.choice(["float32", "bfloat16", "bfloat16", "float16", "float8"]),
                       out_dtype=rng.choice(["float32", "bfloat16", "float16"]))
    V = _log_uniform(rng, 256, 262144)
    B = _log_uniform(rng, 1, max(1, min(4096, (1 << 28) // V)))
    T = rng.choice([0, 0, _log_uniform(rng, 1, 64)]) if B < 512 else 0
    T = min(T, (1 << 28) // (B * V))
    top = rng.choice([0, 1, 5, 20, rng.randint(2, 64)])
    return _rows(op, B, T, V, rng.choice(["float32", "bfloat16", "float16"]), top,
                 temperature=round(rng.uniform(0.5, 2.0), 2), masked=rng.choice([0.0, 0.0, 0.02]))


def _blocks(x, rows):
    """x (R, K) cut into blocks of rows x 128: (R/rows, rows, K/128, 128), zeros where it is not whole."""
    R, K = x.shape
    x = torch.nn.functional.pad(x, (0, -K % BLOCK, 0, -R % rows))
    return x.view(-1, rows, x.shape[1] // BLOCK, BLOCK)


def _quantize(x, rows):
    """The values in 8 bits, (R, K), and the scale of each block, (R/rows, K/128): max |x| / 448, in 32 bits."""
    R, K = x.shape
    b = _blocks(x.float(), rows)
    scale = (b.abs().amax(dim=(1, 3)) / FP8_MAX).clamp(min=SCALE_MIN)
    q = (b / scale[:, None, :, None]).to(torch.float8_e4m3fn)
    q = q.view(torch.uint8).view(b.shape[0] * rows, -1)[:R, :K]
    return q.view(torch.float8_e4m3fn), scale


def _dequantize(q, scale, rows):
    R, K = q.shape
    return (_blocks(q.float(), rows) * scale[:, None, :, None]).view(-1, scale.shape[1] * BLOCK)[:R, :K]


def _padded(q):
    """The same values with rows that begin at multiples of 16 bytes."""
    R, K = q.shape
    out = torch.zeros((R, K + -K % 16), dtype=torch.uint8, device=q.device)
    out[:, :K] = q.view(torch.uint8)
    return out.view(torch.float8_e4m3fn)[:, :K]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        # activations after a norm, some channels far larger than the rest; weights of a trained head's spread
        x = torch.randn((M, K), generator=gen, device="cuda")
        x *= torch.exp(torch.randn((K,), generator=gen, device="cuda"))
        w = torch.randn((N, K), generator=gen, device="cuda").mul_(0.02)
        w, w_scale = _quantize(w, BLOCK)
        state = {"op": "linear", "w": _padded(w), "w_scale": w_scale, "x_scale": None, "out_dtype": DTYPES[case["out_dtype"]]}
        if case["x_dtype"] == "float8":
            x, state["x_scale"] = _quantize(x, 1)
            state["x"] = _padded(x)
        else:
            state["x"] = x.to(DTYPES[case["x_dtype"]])
        return state
    B, T, V = case["B"], case["T"], case["V"]
    shape = (B, T + 1, V) if T else (B, V)
    logits = torch.randn(shape, generator=gen, device="cuda").mul_(2.0)
    # what a confident model gives: a few candidates over a broad floor
    where = torch.randint(0, V, shape[:-1] + (16,), generator=gen, device="cuda")
    logits.scatter_(-1, where, logits.gather(-1, where) + 10.0)
    if case["masked"]:
        logits[..., V - int(V * case["masked"]):] = -math.inf
    logits = logits.to(DTYPES[case["dtype"]])
    tokens = torch.randint(0, V - int(V * case["masked"]), shape[:-1], generator=gen, device="cuda", dtype=torch.int32)
    # every other token is one of the candidates
    tokens = torch.where(torch.rand(shape[:-1], generator=gen, device="cuda") < 0.5, tokens, where[..., 0].int())
    if T:
        logits, tokens = logits[:, :T], tokens[:, 1:].contiguous()
    state = {"op": case["op"], "logits": logits, "tokens": tokens, "temperature": case["temperature"], "top": case["top"]}
    if case["op"] == "gradient":
        state["logits"] = logits.detach().requires_grad_()
        rows = tokens.shape
        state["g"] = torch.randn(rows, generator=gen, device="cuda") / tokens.numel()
        state["h"] = torch.randn(rows, generator=gen, device="cuda").mul_(0.1) / tokens.numel()
        state["a"] = torch.rand(rows + (case["top"],), generator=gen, device="cuda") / (tokens.numel() * max(1, case["top"]))
    return state


def _plain_logprobs(x, tokens, temperature, top):
    """logits (..., V) in 32 bits -> (outputs, what the gradient needs)."""
    V = x.shape[-1]
    at = tokens.long().unsqueeze(-1)
    z = x / temperature
    z = z - z.amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    p = e / total
    entropy = log_total - (p * torch.where(e > 0, z, 0.0)).sum(-1, keepdim=True)
    index = torch.arange(V, device=x.device)
    x_t = x.gather(-1, at)
    rank = 1 + ((x > x_t) | ((x == x_t) & (index < at))).sum(-1)
    # order by the logit, equal ones by the lower index: one whole number of 64 bits for both
    bits = (x + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 32) + (V - 1 - index)
    top_tokens = V - 1 - (order.topk(top, dim=-1).values & 0xFFFFFFFF)
    outputs = ((z.gather(-1, at) - log_total).squeeze(-1), entropy.squeeze(-1), rank.int(),
               z.gather(-1, top_tokens) - log_total, top_tokens.int())
    return outputs, (z, p, log_total, entropy, at, top_tokens)


def run(state):
    if state["op"] == "linear":
        if own:
            import rapid_sampling_amd as sample
            return sample.linear_fp8(state["x"], state["w"], state["w_scale"], x_scale=state["x_scale"],
                                     out_dtype=state["out_dtype"])
        x, x_scale = (state["x"], state["x_scale"]) if state["x_scale"] is not None else _quantize(state["x"], 1)
        return (_dequantize(x, x_scale, 1) @ _dequantize(state["w"], state["w_scale"], BLOCK).T).to(state["out_dtype"])
    logits, tokens, temperature, top = state["logits"], state["tokens"], state["temperature"], state["top"]
    if own:
        import rapid_sampling_amd as sample
        out = sample.token_logprobs(logits, tokens, temperature, top=top)
        if state["op"] == "logprobs":
            return tuple(out)
        wanted, given = (out.logprobs, out.entropy), (state["g"], state["h"])
        if top:
            wanted, given = wanted + (out.top_logprobs,), given + (state["a"],)
        grad, = torch.autograd.grad(wanted, logits, given)
        return out.logprobs.detach(), out.entropy.detach(), out.rank, out.top_logprobs.detach(), out.top_tokens, grad
    out, (z, p, log_total, entropy, at, top_tokens) = _plain_logprobs(logits.detach().float(), tokens, temperature, top)
    if state["op"] == "logprobs":
        return out
    g, h, a = state["g"].unsqueeze(-1), state["h"].unsqueeze(-1), state["a"]
    slope = g + a.sum(-1, keepdim=True) + h * (torch.where(p > 0, z - log_total, 0.0) + entropy)
    grad = (p * -slope).scatter_add_(-1, at, g).scatter_add_(-1, top_tokens, a).div_(temperature)
    return out + (grad.to(logits.dtype),)


def work(case):
    """Inputs read once and outputs written once.  Per logit: the scaling, the exponential, two sums and two comparisons; in
    the gradient the scaling, the exponential and three products and sums."""
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        size = {"float32": 4, "bfloat16": 2, "float16": 2, "float8": 1}
        blocks = -(-K // BLOCK)
        scales = 4 * blocks * (-(-N // BLOCK) + (M if case["x_dtype"] == "float8" else 0))
        return {"bytes": M * K * size[case["x_dtype"]] + N * K + scales + M * N * size[case["out_dtype"]], "flops": 2 * M * N * K}
    rows = case["B"] * max(1, case["T"])
    size = 4 if case["dtype"] == "float32" else 2
    out = rows * (4 + 12 + 8 * case["top"])
    if case["op"] == "logprobs":
        return {"bytes": rows * case["V"] * size + out, "flops": 10 * rows * case["V"]}
    # the gradient needs the row's sums before its first element: the logits are read for both
    return {"bytes": 3 * rows * case["V"] * size + out + rows * (8 + 4 * case["top"]), "flops": 20 * rows * case["V"]}


def _exact_rows(case, state):
    x = state["logits"].detach().double()
    t = state["tokens"].long()[..., None]
    V, T, top = case["V"], case["temperature"], case["top"]
    logp = torch.log_softmax(x / T, dim=-1)
    p = logp.exp()
    weighted = torch.nan_to_num(p * logp, nan=0.0)
    entropy = -weighted.sum(-1)
    x_t = x.gather(-1, t)
    before = torch.arange(V, device=x.device).expand_as(x) < t
    rank = (x > x_t).sum(-1) + ((x == x_t) & before).sum(-1) + 1
    if top:
        ids = torch.cat([torch.sort(rows, dim=-1, descending=True, stable=True).indices[..., :top]
                         for rows in x.view(-1, V).split(1024)]).view(x.shape[:-1] + (top,))
    else:
        ids = torch.empty(x.shape[:-1] + (0,), dtype=torch.long, device=x.device)
    out = (logp.gather(-1, t)[..., 0], entropy, rank.int(), logp.gather(-1, ids), ids.int())
    if case["op"] == "logprobs":
        return out
    # d(logprob_i)/dx_j = ([i = j] - p_j) / T, d(entropy)/dx_j = -p_j (ln p_j + entropy) / T
    g, h, a = state["g"].double(), state["h"].double(), state["a"].double()
    grad = -p * (g + a.sum(-1))[..., None] - (weighted + p * entropy[..., None]) * h[..., None]
    grad.scatter_add_(-1, t, g[..., None])
    grad.scatter_add_(-1, ids, a)
    return out + (grad / T,)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] != "linear":
        state["logits"] = state["logits"].contiguous()
        return _exact_rows(case, state)
    K = case["K"]
    spread = torch.arange(K, device="cuda") // BLOCK
    if state["x_scale"] is None:
        # the roundings to 32 and to 8 bits are the operator's own
        x = state["x"].float()
        peak = torch.zeros((x.shape[0], int(spread[-1]) + 1), device="cuda")
        peak.scatter_reduce_(1, spread.expand_as(x), x.abs(), "amax")
        scale = torch.maximum(peak / FP8_MAX, torch.full_like(peak, SCALE_MIN))
        x = (x / scale[:, spread]).to(torch.float8_e4m3fn)
    else:
        x, scale = state["x"], state["x_scale"]
    x = x.double() * scale.double()[:, spread]
    w = state["w"].double()
    w *= state["w_scale"].double()[torch.arange(case["N"], device="cuda") // BLOCK][:, spread]
    return x @ w.T
