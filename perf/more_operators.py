"""Operators at the two ends of a model's vocabulary table whose time is followed: tokens in (`embedding` and its gradient),
tokens learnt (`linear_cross_entropy` and its gradients) and the head in 8-bit integers (`linear_int8`).

A case is a dict of plain values.  "op" is one of

  "embedding"           rows of the table by token, times a scale; a table in 16 or 32 bits, in 8-bit integers with a scale for each
                        row or in e4m3 with one for each block of 128 x 128
  "embedding_gradient"  the same call under autograd and the gradient of its table
  "loss"                cross entropy of tokens under softmax(x W^T / temperature), and the logarithm of the sum, as a scoring program asks
  "loss_gradient"       the same call under autograd and the gradients of x and W, as a training step makes it
  "linear"              y = x W^T with W in 8-bit integers and a scale for each of its rows; x in 16 or 32 bits, rounded to 8-bit integers
                        within the call with a scale for each row, or (x_dtype "int8") given so

and the rest are sizes:

  M, K, V      tokens or rows of x, columns, rows of the table or weight
  dtype        of table or weight (and of x, for the losses); out_dtype; x_dtype
  padded       share of the tokens that are none (-1)
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
F8 = torch.float8_e4m3fn
BLOCK, SCALE_MIN = 128, 2.0 ** -126


def _embedding(M, K, V, dtype, out_dtype=None, scale=1.0, gradient=False, padded=0.0):
    return {"op": "embedding_gradient" if gradient else "embedding", "M": M, "K": K, "V": V, "dtype": dtype, "out_dtype": out_dtype or dtype,
            "scale": scale, "padded": padded}


def _loss(M, K, V, dtype, temperature=1.0, gradient=True, padded=0.0):
    return {"op": "loss_gradient" if gradient else "loss", "M": M, "K": K, "V": V, "dtype": dtype, "temperature": temperature, "padded": padded}


def _linear(M, K, V, x_dtype="bfloat16", out_dtype="float32"):
    return {"op": "linear", "M": M, "K": K, "V": V, "x_dtype": x_dtype, "out_dtype": out_dtype}


def listed():
    cases = [
        # a serving batch's next tokens, looked up in the table that is the 8-bit head too
        ("embedding_decode", _embedding(64, 4096, 65536, "int8", "bfloat16")),
        # a small training step: an odd number of columns, so that rows begin at any address, some padding, a scaled table
        ("embedding_gradient_ragged", _embedding(385, 1001, 50257, "float16", scale=math.sqrt(1001), gradient=True, padded=0.1)),
        # a training step on rollouts
        ("embedding_gradient_rollouts", _embedding(8192, 4096, 131072, "bfloat16", gradient=True)),
        # one position scored without keeping its logits
        ("loss_one_row", _loss(1, 4096, 65536, "bfloat16", gradient=False)),
        # scoring a batch of prompts
        ("loss_prompts", _loss(2048, 4096, 152064, "bfloat16", gradient=False)),
        # a small training step in float32
        ("loss_gradient_small", _loss(48, 1024, 32768, "float32")),
        # a fine-tuning step: odd sizes, padded texts
        ("loss_gradient_ragged", _loss(385, 2000, 50257, "float16", temperature=1.5, padded=0.2)),
        # a training step on rollouts, at the temperature they were sampled at
        ("loss_gradient_rollouts", _loss(8192, 4096, 131072, "bfloat16", temperature=0.9)),
        # the head of one user's decode loop
        ("linear_one_row", _linear(1, 4096, 65536)),
        # the head of a serving batch
        ("linear_batch", _linear(32, 4096, 131072)),
        # odd sizes: columns that fill no tile, an odd vocabulary
        ("linear_ragged", _linear(77, 2000, 50257, x_dtype="float16", out_dtype="bfloat16")),
        # the head over a prompt, for scoring
        ("linear_prompts", _linear(4096, 4096, 131072, out_dtype="bfloat16")),
    ]
    return [dict(c, name=name) for name, c in cases]


def _log_uniform(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["embedding", "embedding_gradient", "loss", "loss_gradient", "loss_gradient", "linear", "linear"])
    floats = ["float32", "bfloat16", "bfloat16", "float16"]
    K = _log_uniform(rng, 64, 8192)
    if rng.random() < 0.5:
        K += -K % 64
    V = _log_uniform(rng, 512, 152064)
    if op.startswith("embedding"):
        V = min(V, (1 << 29) // K)
        M = _log_uniform(rng, 1, min(32768, (1 << 27) // K))
        dtype = rng.choice(floats if op != "embedding" else floats + ["int8", "float8"])
        out = rng.choice(["float32", "bfloat16", "float16"]) if dtype in ("int8", "float8") else dtype
        return _embedding(M, K, V, dtype, out, scale=rng.choice([1.0, math.sqrt(K), round(rng.uniform(0.1, 10.0), 2)]),
                          gradient=op != "embedding", padded=rng.choice([0.0, 0.0, 0.2]))
    if op == "linear":
        M = _log_uniform(rng, 1, min(8192, max(1, (1 << 40) // (K * V))))
        return _linear(M, K, V, x_dtype=rng.choice(["float32", "bfloat16", "bfloat16", "float16", "int8"]),
                       out_dtype=rng.choice(["float32", "bfloat16", "float16"]))
    dtype = rng.choice(floats)
    most = 1 << (36 if dtype == "float32" else 41)
    M = _log_uniform(rng, 1, min(8192, max(1, most // (K * V))))
    return _loss(M, K, V, dtype, temperature=rng.choice([1.0, round(rng.uniform(0.5, 2.0), 2)]), gradient=op != "loss",
                 padded=rng.choice([0.0, 0.0, 0.2]))


def _quantize_int8(x):
    """8-bit integers and the scale of each row: max |x| / 127, in 32 bits."""
    x = x.float()
    scale = (x.abs().amax(-1) / 127.0).clamp(min=SCALE_MIN)
    return torch.round(x / scale.unsqueeze(-1)).to(torch.int8), scale


def _quantize_fp8(x):
    """e4m3 and the scale of each block of 128 x 128: max |x| / 448, in 32 bits."""
    R, K = x.shape
    b = torch.nn.functional.pad(x, (0, -K % BLOCK, 0, -R % BLOCK))
    b = b.view(-1, BLOCK, b.shape[1] // BLOCK, BLOCK)
    scale = (b.abs().amax(dim=(1, 3)) / 448.0).clamp(min=SCALE_MIN)
    q = (b / scale[:, None, :, None]).to(F8).view(torch.uint8).view(b.shape[0] * BLOCK, -1)
    return q[:R, :K].view(F8), scale


def _padded(q):
    """The same values with rows that begin at multiples of 16 bytes."""
    R, K = q.shape
    out = torch.zeros((R, K + -K % 16), dtype=torch.uint8, device=q.device)
    out[:, :K] = q.view(torch.uint8)
    return out.view(q.dtype)[:, :K]


def _tokens(gen, M, V, padded):
    """What texts hold: a few tokens of every vocabulary make up most of them."""
    u = torch.rand((M,), generator=gen, device="cuda", dtype=torch.float64)
    tokens = (torch.exp(u * math.log(V + 1.0)) - 1.0).long().clamp(max=V - 1)
    tokens = (tokens * 7919) % V                                        # the frequent ones not side by side
    none = torch.rand((M,), generator=gen, device="cuda") < padded
    return torch.where(none, -1, tokens)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, M, K, V = case["op"], case["M"], case["K"], case["V"]
    if op == "linear":
        # activations after a norm, some channels larger than the rest; weights of a trained head's spread
        x = torch.randn((M, K), generator=gen, device="cuda")
        x *= torch.exp(torch.randn((K,), generator=gen, device="cuda").mul_(0.5))
        w, w_scale = _quantize_int8(torch.randn((V, K), generator=gen, device="cuda").mul_(0.02))
        state = {"op": op, "w": _padded(w), "w_scale": w_scale, "x_scale": None, "out_dtype": DTYPES[case["out_dtype"]]}
        if case["x_dtype"] == "int8":
            x, state["x_scale"] = _quantize_int8(x)
            state["x"] = _padded(x)
        else:
            state["x"] = x.to(DTYPES[case["x_dtype"]])
        return state
    tokens = _tokens(gen, M, V, case["padded"])
    if op.startswith("embedding"):
        w = torch.randn((V, K), generator=gen, device="cuda").mul_(0.02)
        state = {"op": op, "tokens": tokens, "scale": case["scale"], "out_dtype": DTYPES[case["out_dtype"]], "w_scale": None}
        if case["dtype"] == "int8":
            w, state["w_scale"] = _quantize_int8(w)
        elif case["dtype"] == "float8":
            w, state["w_scale"] = _quantize_fp8(w)
        state["w"] = _padded(w) if state["w_scale"] is not None else w.to(DTYPES[case["dtype"]])
        if op == "embedding_gradient":
            state["w"].requires_grad_()
            state["g"] = torch.randn((M, K), generator=gen, device="cuda").div_(M).to(state["out_dtype"])
        return state
    dtype = DTYPES[case["dtype"]]
    w = torch.randn((V, K), generator=gen, device="cuda").mul_(2.0 / math.sqrt(K))
    x = torch.randn((M, K), generator=gen, device="cuda")
    # what a trained model gives: most tokens are among its likely ones
    sure = torch.rand((M, 1), generator=gen, device="cuda").mul_(2.5)
    x += w[tokens.clamp(min=0)] * sure
    state = {"op": op, "tokens": tokens, "x": x.to(dtype), "w": w.to(dtype), "temperature": case["temperature"]}
    if op == "loss_gradient":
        state["x"].requires_grad_()
        state["w"].requires_grad_()
        state["g"] = torch.randn((M,), generator=gen, device="cuda").mul_(0.5).add_(1.0).div_(M)
        state["h"] = torch.randn((M,), generator=gen, device="cuda").mul_(0.01 / M)
    return state


def _own(state):
    import rapid_sampling_amd as sample
    op = state["op"]
    if op == "linear":
        return sample.linear_int8(state["x"], state["w"], state["w_scale"], x_scale=state["x_scale"], out_dtype=state["out_dtype"])
    if op.startswith("embedding"):
        y = sample.embedding(state["tokens"], state["w"], state["scale"], weight_scale=state["w_scale"], out_dtype=state["out_dtype"])
        if op == "embedding":
            return y
        return y.detach(), torch.autograd.grad(y, state["w"], state["g"])[0]
    out = sample.linear_cross_entropy(state["x"], state["w"], state["tokens"], state["temperature"])
    if op == "loss":
        return tuple(out)
    grads = torch.autograd.grad((out.loss, out.logsumexp), (state["x"], state["w"]), (state["g"], state["h"]))
    return (out.loss.detach(), out.logsumexp.detach()) + grads


def _plain_rows(q, w_scale, tokens):
    """Rows of the table in 32 bits, zeros where there is no token."""
    there = tokens >= 0
    at = tokens.clamp(min=0)
    rows = q.detach()[at].float()
    if q.dtype == torch.int8:
        rows = rows * w_scale[at].unsqueeze(-1)
    elif q.dtype == F8:
        scale = w_scale[at // BLOCK].repeat_interleave(BLOCK, dim=-1)[:, :q.shape[1]]
        rows = rows * scale
    return torch.where(there.unsqueeze(-1), rows, 0.0)


def run(state):
    if own:
        return _own(state)
    op = state["op"]
    if op == "linear":
        x, x_scale = (state["x"], state["x_scale"]) if state["x_scale"] is not None else _quantize_int8(state["x"])
        y = x.float() @ state["w"].float().T
        return (y * (x_scale.unsqueeze(-1) * state["w_scale"])).to(state["out_dtype"])
    tokens = state["tokens"]
    there = tokens >= 0
    if op.startswith("embedding"):
        y = (_plain_rows(state["w"], state["w_scale"], tokens) * state["scale"]).to(state["out_dtype"])
        if op == "embedding":
            return y
        w = state["w"]
        order = torch.argsort(torch.where(there, tokens, w.shape[0]), stable=True)
        grad = torch.zeros((w.shape[0] + 1, w.shape[1]), device=w.device)
        grad.index_add_(0, torch.where(there, tokens, w.shape[0])[order], state["g"][order].float())
        return y, (grad[:-1] * state["scale"]).to(w.dtype)
    x, w, inv = state["x"].detach().float(), state["w"].detach().float(), 1.0 / state["temperature"]
    at = tokens.clamp(min=0).unsqueeze(-1)
    z = (x @ w.T).mul_(inv)
    m = z.amax(-1, keepdim=True)
    z_t = z.gather(-1, at)
    p = z.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    lse = torch.log(total) + m
    loss = torch.where(there, (lse - z_t).squeeze(-1), 0.0)
    lse = lse.squeeze(-1)
    if op == "loss":
        return loss, lse
    g = torch.where(there, state["g"], 0.0).unsqueeze(-1)
    grad = p.div_(total).mul_(g + state["h"].unsqueeze(-1)).scatter_add_(-1, at, -g).mul_(inv)
    return loss, lse, (grad @ w).to(state["x"].dtype), (grad.T @ x).to(state["w"].dtype)


def work(case):
    """Inputs read once and outputs written once.  Of a table's rows only those that are named are read; a gradient of a table is written whole.
    Losses: the product of x and W, and two more of its size for their gradients."""
    size = {"float32": 4, "bfloat16": 2, "float16": 2, "int8": 1, "float8": 1}
    op, M, K, V = case["op"], case["M"], case["K"], case["V"]
    if op == "linear":
        scales = 4 * V + (4 * M if case["x_dtype"] == "int8" else 0)
        return {"bytes": M * K * size[case["x_dtype"]] + V * K + scales + M * V * size[case["out_dtype"]], "flops": 2 * M * V * K}
    s = size[case["dtype"]]
    if op.startswith("embedding"):
        out = size[case["out_dtype"]]
        read = {"bytes": 8 * M + min(M, V) * K * s + M * K * out, "flops": M * K}
        if op == "embedding":
            return read
        return {"bytes": read["bytes"] + M * K * out + V * K * s, "flops": 3 * M * K}
    read = (M + V) * K * s + 8 * M + 8 * M
    if op == "loss":
        return {"bytes": read, "flops": 2 * M * V * K}
    return {"bytes": read + 8 * M + (M + V) * K * s, "flops": 6 * M * V * K}


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        x, x_scale = state["x"], state["x_scale"]
        if x_scale is None:
            # the roundings to 32 bits and to integers are the operator's own
            x = x.float()
            x_scale = torch.maximum(x.abs().max(dim=1).values / 127.0, torch.full((x.shape[0],), SCALE_MIN, device="cuda"))
            x = (x / x_scale[:, None]).round()
        y = x.double() @ state["w"].double().T
        return y * x_scale.double()[:, None] * state["w_scale"].double()[None, :]
    t, w = state["tokens"], state["w"].detach()
    real = (t >= 0).double()[:, None]
    index = t.clamp(min=0)
    if op.startswith("embedding"):
        rows = w[index].double()
        if w.dtype == torch.int8:
            rows *= state["w_scale"].double()[index][:, None]
        elif w.dtype == F8:
            columns = torch.arange(case["K"], device="cuda") // BLOCK
            rows *= state["w_scale"].double()[index // BLOCK][:, columns]
        y = rows * real * case["scale"]
        if op == "embedding":
            return y
        grad = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
        grad.index_put_((index,), state["g"].double() * real * case["scale"], accumulate=True)
        return y, grad
    x, w = state["x"].detach().double(), w.double()
    logits = (x @ w.T) / case["temperature"]
    lse = torch.logsumexp(logits, dim=-1)
    loss = (lse - logits.gather(-1, index[:, None])[:, 0]) * real[:, 0]
    if op == "loss":
        return loss, lse
    g, h = state["g"].double() * real[:, 0], state["h"].double()
    # d(loss_i)/dz_j = p_j - [i = j], d(lse)/dz_j = p_j
    dz = torch.exp(logits - lse[:, None])
    del logits
    dz *= (g + h)[:, None]
    dz[torch.arange(case["M"], device="cuda"), index] -= g
    dz /= case["temperature"]
    return loss, lse, dz @ w, dz.T @ x
