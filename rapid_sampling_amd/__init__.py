"""MI355X-native batched token sampler: temperature, top-k, top-p, presence /
repetition penalties with in-place decay.

Drop-in for the Python API of the reference module (`sample` in
/root/reference/example.py:13-33; bound at /root/reference/sampling.cpp:5-8):

    import rapid_sampling_amd as sample
    states  = sample.setup_rand(0, B)
    tokens  = sample.batch_sampling_temperature_topk_topp(logits, states, temperature, top_k, top_p)
    tokens  = sample.batch_sampling_repetition_temperature_topk_topp(
                  logits, penalties, states, presence_penalty, repetition_penalty,
                  penalty_decay, temperature, top_k, top_p)

Beyond the reference: keyword names, `uniforms=` (injected draws, for tests),
`accept_half=True` (bfloat16 / float16 logits read as they are; by default any
type but float32 raises the reference's error), `reserve_workspace(B, V)`
(allocates the current stream's workspaces ahead of time: required before the
calls are captured into a HIP graph; any V, and `operators=False` leaves out the
12.6 MB of the functions next to the sampler), `workspace_status()` (synchronises and
returns the error word of the current stream's workspace), `set_wait_limit` and
`reset_routing()` (forgets what the stream's calls have learnt about which
kernel suits the workload; for measurements that change workload on one stream).
A call whose kernel gave up waiting for its peers raises RuntimeError on the
next call on that stream at the latest.

Next to the sampler:

    y = sample.linear_fp8(hidden, weight, weight_scale)      # an 8-bit head: logits from hidden states
    out = sample.token_logprobs(logits, tokens, temperature, top=5)

`token_logprobs` gives, for each row of (V,), (B, V) or (B, T, V) logits (float32, bfloat16 or float16; any V up
to 1048576, rows at any stride) and its token, the token's log probability at that temperature, the row's entropy,
the token's rank (1: the likeliest) and the `top` (up to 64) likeliest alternatives, equal logits by the lower token.
A negative token is none (padding): log probability 0, rank 0.  It can be differentiated (once, in reverse mode) by its logits.
`linear_fp8(x, weight, weight_scale)` is x @ weight.T for a float8_e4m3fn weight with a float32 scale for each block of
128 x 128; x in float32, bfloat16 or float16 is rounded to 8 bits within the call, with a scale for each 128 values of a
row, or is given so with x_scale=.  `quantize_fp8(x)` makes such values and scales, `quantize_fp8(w, block_rows=128)`
those of a weight.  Neither has a gradient, and what asks for one is refused; that of x, in 8 bits as well, is the same product with the
transposed weight, whose blocks are the weight's own, in rows that begin at multiples of 16 bytes whatever N is:

    N, K = weight.shape
    transposed = torch.zeros((K, N + -N % 16), dtype=torch.uint8, device=weight.device)
    transposed[:, :N] = weight.view(torch.uint8).t()
    transposed = transposed.view(torch.float8_e4m3fn)[:, :N]
    grad_x = sample.linear_fp8(grad, transposed, weight_scale.t().contiguous())

The functions live in the compiled extension `_sample` (host layer in
csrc/sampling.cpp, kernels in csrc/rs_*.hip and csrc/rs_*.h behind the C ABI of
include/rapid_sampling.h).  There is no Python or CPU fallback: without the
built extension the import fails.
"""
import os as _os
from typing import NamedTuple as _NamedTuple

import torch as _torch  # noqa: F401  (loads libtorch before the extension)

_HERE = _os.path.dirname(_os.path.abspath(__file__))

try:
    from . import _sample
except ImportError as _e:  # pragma: no cover - exercised only on an unbuilt tree
    raise ImportError(
        "rapid_sampling_amd: the compiled extension is missing or does not load (%s). "
        "Build it in-tree with `python rapid_sampling_amd/build.py`." % (_e,)
    ) from _e

setup_rand = _sample.setup_rand
batch_sampling_temperature_topk_topp = _sample.batch_sampling_temperature_topk_topp
batch_sampling_repetition_temperature_topk_topp = _sample.batch_sampling_repetition_temperature_topk_topp
batch_sampling_debug = _sample.batch_sampling_debug
floor_read = _sample.floor_read
reserve_workspace = _sample.reserve_workspace
workspace_status = _sample.workspace_status
set_wait_limit = _sample.set_wait_limit
reset_routing = _sample.reset_routing
quantize_fp8 = _sample.quantize_fp8
linear_fp8 = _sample.linear_fp8
LOGPROBS_TOP_MAX = _sample.LOGPROBS_TOP_MAX
STATE_BYTES_PER_ROW = _sample.STATE_BYTES_PER_ROW
DIAG_BYTES = _sample.DIAG_BYTES


class TokenLogprobs(_NamedTuple):
    """What token_logprobs returns, each of the tokens' shape (the alternatives with one axis more)."""
    logprobs: _torch.Tensor        # float32
    entropy: _torch.Tensor         # float32, in nats
    rank: _torch.Tensor            # int32, from 1
    top_logprobs: _torch.Tensor    # float32, likeliest first
    top_tokens: _torch.Tensor      # int32


def token_logprobs(logits, tokens, temperature=1.0, *, top=0):
    """Log probabilities of `tokens` (int32 or int64) under softmax(logits / temperature), with the rows' entropy, the tokens'
    ranks and the `top` likeliest alternatives: a TokenLogprobs.  See the module's docstring."""
    return TokenLogprobs(*_sample.token_logprobs(logits, tokens, temperature, top=top))


KERNEL_LIBRARY = _os.path.join(_HERE, "librapid_sampling_hip.so")

__all__ = [
    "setup_rand",
    "batch_sampling_temperature_topk_topp",
    "batch_sampling_repetition_temperature_topk_topp",
    "batch_sampling_debug",
    "token_logprobs",
    "TokenLogprobs",
    "quantize_fp8",
    "linear_fp8",
    "floor_read",
    "reserve_workspace",
    "workspace_status",
    "set_wait_limit",
    "reset_routing",
    "LOGPROBS_TOP_MAX",
    "STATE_BYTES_PER_ROW",
    "DIAG_BYTES",
    "KERNEL_LIBRARY",
]
