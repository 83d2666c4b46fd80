"""token_logprobs and its gradient against the formulas in 64 bits.

With eps = 2^-24 a term's argument z = (x - m) c carries two roundings and c's own, its exponential one unit in the last
place, and a sum's longest chain is of V / 1024 + 32 additions (four logits and more are added up before they join a thread's
sum, a workgroup of 256 joins in 8 steps): every sum is within eps (64 + V / 1024 + 8 |z|) of itself, |z| the arguments that
weigh, and so are the results, with log(S), z_t and H as their scale."""
import math

import pytest
import torch

EPS = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}       # half a unit in the last place
LEAST = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}
INF = math.inf

gpu = pytest.mark.gpu


def formulas(x, tokens, temperature, top):
    """(logprobs, entropy, rank, top_logprobs, top_tokens) of x (R, V) and tokens (R,), on the CPU in 64 bits."""
    x, V = x.detach().cpu().double(), x.shape[-1]
    z = x / temperature
    m = z.amax(-1, keepdim=True)
    empty = m == -INF
    d = torch.where(empty, -INF, z - m)
    e = torch.exp(d)
    s = e.sum(-1, keepdim=True)
    lp = torch.where(empty, -INF, d - torch.log(s))
    entropy = -(torch.where(e > 0, e * lp, 0.0 * e) / s).sum(-1)
    entropy = torch.where(empty.squeeze(-1), 0.0, entropy)
    order = [sorted(range(V), key=lambda i: (math.isnan(r[i]), -r[i] if not math.isnan(r[i]) else 0.0, i)) for r in x.tolist()]
    t = tokens.cpu().tolist()
    rank = [o.index(i) + 1 if 0 <= i < V else 0 for o, i in zip(order, t)]
    ids = torch.tensor([o[:top] for o in order], dtype=torch.long).reshape(len(t), top)
    given = [lp[r, i].item() if 0 <= i < V else (0.0 if i < 0 else math.nan) for r, i in enumerate(t)]
    return torch.tensor(given, dtype=torch.float64), entropy, torch.tensor(rank), lp.gather(1, ids), ids


def gradient(x, tokens, temperature, g, h, a, ids):
    x = x.detach().cpu().double()
    lp = torch.log_softmax(x / temperature, -1)
    p = lp.exp()
    q = torch.where(p > 0, p * lp, 0.0 * p)
    out = -p * (g + a.sum(-1))[:, None] - h[:, None] * (q - p * q.sum(-1, keepdim=True))
    out.scatter_add_(1, tokens.cpu().long()[:, None], g[:, None])
    out.scatter_add_(1, ids, a)
    return out / temperature


def near(got, want, scale, V, what):
    got, want = got.detach().cpu().double(), want.float().double()
    assert torch.equal(got.isnan(), want.isnan()), what
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), what
    ok = ~(inf | want.isnan())
    bound = EPS * (64 + V / 1024 + 8 * 40) * (1 + scale.double().expand_as(want)[ok].abs())
    off = (got - want)[ok].abs()
    assert (off <= bound).all(), (what, off.max().item(), bound.min().item())


def check(logits, tokens, temperature=1.0, top=0, rows=None):
    import rapid_sampling_amd as sample
    V = logits.shape[-1]
    out = sample.token_logprobs(logits, tokens, temperature, top=top)
    torch.cuda.synchronize()
    shape = logits.shape[:-1]
    assert out.logprobs.shape == out.entropy.shape == out.rank.shape == shape and out.top_tokens.shape == shape + (top,)
    want = formulas(logits.reshape(-1, V), tokens.reshape(-1), temperature, top)
    flat = [o.reshape((tokens.numel(),) + o.shape[len(shape):]) for o in out]
    near(flat[0], want[0], want[0].nan_to_num(0, 0, 0), V, "logprobs")
    near(flat[1], want[1], torch.full_like(want[1], math.log(V)), V, "entropy")
    assert flat[2].cpu().tolist() == want[2].tolist()
    assert flat[4].cpu().tolist() == want[4].tolist()
    near(flat[3], want[3], want[3].nan_to_num(0, 0, 0), V, "top_logprobs")
    return out


def make(rows, V, dtype, seed, scale=3.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, V), generator=gen) * scale).to(DTYPES[dtype]).cuda()
    return x, torch.randint(0, V, (rows,), generator=gen).cuda()


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [1, 2, 3, 7, 8, 9, 63, 255, 1023, 1024, 1025, 4099, 8192, 20001])
def test_sizes(V, dtype):
    print("sizes", V, dtype, flush=True)
    for rows, top in ((1, min(V, 5)), (3, min(V, 64)), (2, 0)):
        x, t = make(rows, V, dtype, V + rows)
        check(x, t, 0.8, top)


@gpu
@pytest.mark.parametrize("rows", [1, 5, 200, 1100, 3000])
def test_rows_split_and_whole(rows):
    """Few rows are split over workgroups, many are not."""
    print("rows", rows, flush=True)
    V = 9001 if rows < 1000 else 601
    x, t = make(rows, V, "bf16", rows)
    check(x, t.int(), 1.3, 7)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [1, 7, 64, 300, 2049, 5000])
def test_many_short_rows(V, dtype):
    """Rows that a wave does by itself, masked ones among them."""
    print("short rows", V, dtype, flush=True)
    x, t = make(2300, V, dtype, V, scale=2.0)
    if V > 60:
        x[::7, V // 3:] = -INF
        x[::11] = torch.finfo(x.dtype).min
        x[::13] = -INF
        x[5, :] = 1.0
    pick = torch.cat([torch.arange(40), torch.arange(2260, 2300)]).cuda()
    import rapid_sampling_amd as sample
    for top in (0, min(V, 3), min(V, 32), min(V, 64)):
        out = sample.token_logprobs(x, t, 0.9, top=top)
        some = check(x[pick], t[pick], 0.9, top)                      # (fewer rows: by workgroups)
        want = formulas(x[pick], t[pick], 0.9, top)
        assert out.rank[pick].tolist() == want[2].tolist() and out.top_tokens[pick].tolist() == want[4].tolist()
        for a, b in zip((out.logprobs, out.entropy, out.top_logprobs), (some.logprobs, some.entropy, some.top_logprobs)):
            near(a[pick], b.cpu(), b.cpu().double().nan_to_num(0, 0, 0), V, "short rows")


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_long_rows(dtype):
    x, t = make(2, 131072 + 5, dtype, 1)
    check(x, t, 1.0, 20)
    x, t = make(1, 1048576, dtype, 2)
    check(x, t, 0.5, 64)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_positions_slices_and_strides(dtype):
    import rapid_sampling_amd as sample
    gen = torch.Generator().manual_seed(5)
    full = (torch.randn((3, 9, 1003), generator=gen) * 3).to(DTYPES[dtype]).cuda()
    ids = torch.randint(0, 997, (3, 9), generator=gen).cuda()
    check(full[:, :-1], ids[:, 1:], 1.0, 3)                        # the usual shift: neither is contiguous
    check(full[..., 3:1000], ids, 1.0, 3)                          # rows that begin anywhere
    check(full.transpose(0, 1), ids.t(), 1.0, 2)
    check(full[0, 0], ids[0, 0], 1.0, 2)                           # (V,) and ()
    check(full[:, 2], ids[:, 2].int(), 1.0, 2)
    one = full[1, 1].expand(4, 5, 1003)                            # one row for all
    check(one, ids[:1, :5].expand(4, 5), 1.0, 2)
    empty = sample.token_logprobs(full[:0], ids[:0], top=4)
    assert empty.top_tokens.shape == (0, 9, 4) and empty.logprobs.shape == (0, 9)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [100, 5000, 40000])
def test_masks(V, dtype):
    print("masks", V, dtype, flush=True)
    x, t = make(9, V, dtype, 3)
    low = torch.finfo(x.dtype).min
    x[0, V // 2:] = -INF
    x[1, :-1] = -INF                                               # one token left
    x[2] = -INF                                                    # none left
    x[3] = low                                                     # none left, by the lowest value: uniform
    x[4, 10:] = low
    x[5, 3] = -x[5, 3].abs() * 0 - 0.0                             # a negative zero among zeros
    x[5, 4:60] = 0.0
    x[6, 1::2] = -INF
    x[7, 1:] = low
    x[7, 0] = torch.finfo(x.dtype).max
    x[8, ::3] = -INF
    t[1], t[2], t[4], t[5], t[6] = V - 1, 5, 50, 40, 1
    check(x, t, 1.0, 20)
    check(x, t, 0.01, 5)


@gpu
@pytest.mark.parametrize("V", [50, 3000])
def test_values_that_are_no_numbers(V):
    x, t = make(6, V, "f32", 4)
    x[0, 7] = math.nan
    x[1, 7] = INF
    x[2, 7], t[2] = INF, 7
    x[3, 9], t[3] = math.nan, 9
    x[3, 2] = math.nan
    x[4] = math.nan
    x[5, ::2], t[5] = -math.nan, 11
    import rapid_sampling_amd as sample
    out = sample.token_logprobs(x, t, top=V if V <= 64 else 30)
    want = formulas(x, t, 1.0, V if V <= 64 else 30)
    assert out.logprobs.isnan().all() and out.entropy.isnan().all() and out.top_logprobs.isnan().all()
    assert out.rank.tolist() == want[2].tolist() and out.top_tokens.tolist() == want[4].tolist()


@gpu
def test_tokens_that_are_none():
    x, t = make(4, 777, "f32", 6)
    t[0], t[1], t[2] = -100, 777, 1 << 40
    out = check(x, t, 1.0, 3)
    assert out.logprobs[0].item() == 0.0 and out.logprobs[1:3].isnan().all() and out.rank[:3].tolist() == [0, 0, 0]


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows", [2, 1030, 2100])
def test_rows_whose_alternatives_are_hard_to_find(rows, dtype):
    """Equal logits by the thousand, sorted rows, and large logits that all fall to one thread of the pass."""
    V = 20000 if rows == 2 else 2100
    gen = torch.Generator().manual_seed(8)
    kinds = [torch.zeros(V), torch.arange(V) / 64.0, -torch.arange(V) / 64.0, torch.randint(0, 2, (V,), generator=gen).float(),
             torch.where(torch.arange(V) // 8 % 256 == 5, 5.0, 0.0) + torch.rand(V, generator=gen),
             torch.where(torch.arange(V) // 4 % 256 == 77, 5.0, -5.0), torch.full((V,), -INF).index_fill_(0, torch.arange(V - 9, V), 1.0)]
    for n, row in enumerate(kinds):
        print("hard", rows, dtype, n, flush=True)
        x = row.to(DTYPES[dtype]).cuda().expand(rows, V)
        t = torch.tensor([V // 2, V - 1]).cuda()
        for top in (1, 30, 64):
            import rapid_sampling_amd as sample
            out = sample.token_logprobs(x, t[torch.arange(rows, device="cuda") % 2], top=top)
            want = formulas(x[:2], t, 1.0, top)
            for r in (0, 1, rows - 2, rows - 1):
                assert out.top_tokens[r].tolist() == want[4][r % 2].tolist(), (n, top)
                assert out.rank[r].item() == want[2][r % 2].item(), (n, top)


@gpu
def test_largest_of_one_thread_only():
    """More candidates than the list holds: one thread of the pass has 512 of the row's largest logits."""
    V = 131072
    x = torch.randn(V, generator=torch.Generator().manual_seed(3))
    x = x + torch.where(torch.arange(V) // 4 % 256 == 5, 20.0, 0.0)
    check(x.cuda().expand(1, V), torch.tensor([20]).cuda(), 1.0, 64)
    check(x.cuda().expand(1100, V)[:2], torch.tensor([20, 21]).cuda(), 1.0, 64)


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V,top", [(1, 1), (5, 2), (1000, 0), (1027, 64), (8195, 3), (33000, 20)])
def test_gradient(V, top, dtype):
    import rapid_sampling_amd as sample
    print("gradient", V, top, dtype, flush=True)
    rows, T = 5, 0.7
    x, t = make(rows, V, dtype, V)
    if V > 500:
        x[1, V // 2:] = -INF
        x[2, 3:] = torch.finfo(x.dtype).min
        t[1], t[2] = 4, 1
        t[3] = x[3].float().argmax()                               # the token is an alternative too
    x.requires_grad_()
    gen = torch.Generator().manual_seed(1)
    g, h, a = torch.randn(rows, generator=gen), torch.randn(rows, generator=gen), torch.randn((rows, top), generator=gen)
    out = sample.token_logprobs(x, t, T, top=top)
    got, = torch.autograd.grad((out.logprobs, out.entropy, out.top_logprobs), x, (g.cuda(), h.cuda(), a.cuda()))
    assert got.dtype == x.dtype and got.shape == x.shape
    g, h, a = g.double(), h.double(), a.double()
    ids = out.top_tokens.cpu().long()
    want = gradient(x, t, T, g, h, a, ids)
    lp = torch.log_softmax(x.detach().cpu().double() / T, -1)
    p, z = lp.exp(), lp.clamp(min=-200).abs()
    size = p * (g.abs() + a.abs().sum(-1) + h.abs() * (math.log(V) + 1))[:, None] + p * h.abs()[:, None] * z
    size.scatter_add_(1, t.cpu()[:, None], g.abs()[:, None])
    size.scatter_add_(1, ids, a.abs())
    bound = EPS * (64 + V / 1024 + 8 * 40 + 8 * z) * size / T + UNIT[x.dtype] * want.abs() * 1.01 + LEAST[x.dtype]
    off = (got.cpu().double() - want).abs()
    assert (off <= bound).all(), (off / bound).max().item()


@gpu
def test_gradient_against_differences():
    """d/dx_i of sum g logprob + h entropy + sum a top_logprobs, by central differences of the formulas in 64 bits: their error is
    of the order of step^2 = 1e-10 and of 1e-16 / step = 1e-11; the gradient's own bound is eps 400 = 2.4e-5."""
    import rapid_sampling_amd as sample
    V, T, step = 37, 0.9, 1e-5
    x, t = make(1, V, "f32", 12, scale=1.0)
    x.requires_grad_()
    out = sample.token_logprobs(x, t, T, top=3)
    ids = out.top_tokens.cpu().long()[0]
    (0.7 * out.logprobs.sum() - 0.4 * out.entropy.sum() + 0.3 * out.top_logprobs.sum()).backward()

    def value(v):
        lp = torch.log_softmax(v / T, -1)
        return 0.7 * lp[t.cpu()[0]] + 0.4 * (lp.exp() * lp).sum() + 0.3 * lp[ids].sum()
    v = x.detach().cpu().double()[0]
    for i in range(V):
        d = torch.zeros(V, dtype=torch.float64)
        d[i] = step
        assert abs((value(v + d) - value(v - d)).item() / (2 * step) - x.grad[0, i].item()) < 2.5e-5


@gpu
def test_gradient_of_what_is_used():
    """Outputs left out, gradients that are broadcast, rows that are shared, tokens that are none, rows that are empty."""
    import rapid_sampling_amd as sample
    x, t = make(4, 501, "f32", 20)
    x[2] = -INF
    t[1] = -1
    z, one = torch.zeros(4, dtype=torch.float64), torch.ones(4, dtype=torch.float64)
    none = torch.zeros((4, 0), dtype=torch.float64)
    ids = torch.zeros((4, 0), dtype=torch.long)
    keep = [0, 1, 3]

    def grad(f, y=None):
        y = (x if y is None else y).detach().requires_grad_()
        f(sample.token_logprobs(y, t)).backward()
        return y.grad.cpu().double()
    bound = EPS * 400 * 10
    got = grad(lambda o: o.logprobs.sum())
    want = gradient(x, t.clamp(min=0), 1.0, one * torch.tensor([1., 0, 1, 1]), z, none, ids)
    assert (got - want)[keep].abs().max() < bound and (got[2] == 0).all() and (got[1] == 0).all()
    got = grad(lambda o: o.entropy.sum())
    want = gradient(x, t.clamp(min=0), 1.0, z, one, none, ids)
    assert (got - want)[keep].abs().max() < bound and (got[2] == 0).all()
    # a shared row's gradient is the sum of its uses'
    y = x[0].detach().requires_grad_()
    sample.token_logprobs(y.expand(4, 501), t.clamp(min=0)).logprobs.sum().backward()
    want = gradient(x[:1].expand(4, 501), t.clamp(min=0), 1.0, one, z, none, ids).sum(0)
    assert (y.grad.cpu().double() - want).abs().max() < 4 * bound
    # a slice of a larger tensor
    y = torch.randn((2, 3, 501), device="cuda").requires_grad_()
    s = torch.randint(0, 501, (2, 2), device="cuda")
    sample.token_logprobs(y[:, :-1], s).logprobs.sum().backward()
    assert (y.grad[:, -1] == 0).all() and (y.grad[:, 0].abs().sum() > 0)
    # nothing asked for: nothing is kept
    with torch.no_grad():
        assert not sample.token_logprobs(y, torch.zeros((2, 3), dtype=torch.long, device="cuda")).logprobs.requires_grad
    # a second derivative is refused, not zero
    y = x.detach().requires_grad_()
    d, = torch.autograd.grad(sample.token_logprobs(y, t).entropy.sum(), y, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        d.sum().backward()
    out = sample.token_logprobs(y, t, top=2)
    assert not out.rank.requires_grad and not out.top_tokens.requires_grad and out.top_logprobs.requires_grad


@gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_gradient_of_a_row_whose_token_is_outside(dtype):
    """The entropy and the alternatives of a row do not depend on its token, and neither do their gradients; the log probability of a
    token that is outside the vocabulary is NaN, and its gradient with it."""
    import rapid_sampling_amd as sample
    V, T = 3001, 0.8
    x, t = make(4, V, dtype, 21)
    t[1], t[2] = V, 1 << 40
    keep = [0, 3]
    z = torch.zeros(4, dtype=torch.float64)
    h, a = torch.tensor([0.5, -1.0, 2.0, 1.0]), torch.randn((4, 5), generator=torch.Generator().manual_seed(2))

    def grad(f):
        y = x.detach().requires_grad_()
        out = sample.token_logprobs(y, t, T, top=5)
        f(out).backward()
        return y.grad.cpu().double(), out.top_tokens.cpu().long()
    within = t.clamp(max=V - 1)
    got, ids = grad(lambda o: (o.entropy * h.cuda()).sum())
    want = gradient(x, within, T, z, h.double(), torch.zeros((4, 5), dtype=torch.float64), ids)
    limit = lambda want: EPS * 400 * 20 + UNIT[x.dtype] * want.abs() * 1.01 + LEAST[x.dtype]
    assert ((got - want).abs() <= limit(want)).all()
    got, ids = grad(lambda o: (o.top_logprobs * a.cuda()).sum())
    want = gradient(x, within, T, z, z, a.double(), ids)
    assert ((got - want).abs() <= limit(want)).all()
    got, ids = grad(lambda o: o.logprobs[keep].sum() + (o.entropy * h.cuda()).sum())
    assert got[1:3].isnan().all() and not got[keep].isnan().any()


@gpu
def test_streams_and_graphs():
    import rapid_sampling_amd as sample
    x, t = make(3, 50001, "f32", 30)
    want = sample.token_logprobs(x, t, top=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sample.token_logprobs(x, t, top=5)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.cuda.stream(side):
        sample.reserve_workspace(3, 50004)
        graph = torch.cuda.CUDAGraph()
        y = x.clone()
        with torch.cuda.graph(graph, stream=side):
            held = sample.token_logprobs(y, t, top=5)
    for seed in range(4):
        fresh, _ = make(3, 50001, "f32", 40 + seed)
        y.copy_(fresh)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = sample.token_logprobs(fresh, t, top=5)
        assert all(torch.equal(a, b) for a, b in zip(held, want)), seed


@gpu
def test_more_elements_than_32_bits_count():
    """The last rows of more than 2^31 logits, against the same rows by themselves; their gradient too."""
    import rapid_sampling_amd as sample
    V, rows = 1048576, 2060
    x = torch.zeros((rows, V), dtype=torch.bfloat16, device="cuda")
    last = slice(rows - 3, rows)
    x[last] = make(3, V, "bf16", 77)[0]
    t = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(1)).cuda()
    want = check(x[last], t[last], 1.0, 5)
    got = sample.token_logprobs(x, t, top=5)
    for a, b in zip(got, want):
        assert torch.equal(a[last], b) if not a.is_floating_point() else torch.allclose(a[last], b, rtol=0, atol=EPS * (64 + V / 1024) * 20)
    part = x[last].clone().requires_grad_()
    sample.token_logprobs(part, t[last]).logprobs.sum().backward()
    x.requires_grad_()
    sample.token_logprobs(x, t).logprobs.sum().backward()
    assert torch.equal(x.grad[last], part.grad)


def test_refusals():
    import rapid_sampling_amd as sample
    x, t = torch.zeros((2, 8)), torch.zeros(2, dtype=torch.long)
    bad = [((x.double(), t), {}, "float32"), ((x, t.float()), {}, "int32"), ((x, t[:1]), {}, "shape"), ((x[None, None], t), {}, "shape"),
           ((x, t, 0.0), {}, "Temperature"), ((x, t, math.nan), {}, "Temperature"), ((x, t), {"top": 9}, "top"), ((x, t), {"top": -1}, "top"),
           ((torch.zeros((2, 100)), t), {"top": 65}, "top"), ((x[:, :0], t), {}, "Vocabulary"), ((x, t), {}, "GPU"),
           ((torch.zeros(()), t), {}, "shape")]
    for args, kw, text in bad:
        with pytest.raises(ValueError, match=text):
            sample.token_logprobs(*args, **kw)


def test_refusals_of_the_c_abi():
    import ctypes as C

    from tests import capi
    L = capi.lib()
    size = C.c_size_t
    L.rs_logprobs_workspace_bytes.restype = size
    n = L.rs_logprobs_workspace_bytes()
    p, i32, i64 = C.c_void_p, C.c_int32, C.c_int64
    L.rs_token_logprobs.argtypes = [p, i32, i64, i64, p, i32, i64, i64, i32, i32, i32, C.c_double, i32] + [p] * 6 + [p, size, p]
    L.rs_token_logprobs_backward.argtypes = [p, i32, i64, i64, p, i32, i64, i64, i32, i32, i32, C.c_double, i32, p, p, p, i32, p, i32, p, i32, p, p]

    def call(logits=256, dtype=0, tokens=256, wide=0, B=1, T=1, V=8, temp=1.0, top=0, ids=256, stats=0, ws=256, ws_bytes=n):
        return L.rs_token_logprobs(logits, dtype, V, V, tokens, wide, 1, 1, B, T, V, temp, top, 256, 256, 256, ids, ids, stats, ws, ws_bytes, None)
    assert call(V=0) == call(V=1048577) == -1 and call(B=0) == call(T=0) == call(B=65536, T=65536) == -2
    assert call(temp=0.0) == call(temp=math.nan) == -3 and call(logits=None) == call(tokens=None) == call(ws=None) == call(top=1, ids=None) == -4
    assert call(ws_bytes=n - 1) == call(ws=8) == -5 and call(logits=257) == call(tokens=258) == call(wide=1, tokens=260) == call(stats=8) == -6
    assert call(dtype=3) == call(top=9) == call(top=65, V=100) == call(wide=2) == -7

    def back(stats=256, ids=256, gs=1, a=None, out=256, top=0):
        return L.rs_token_logprobs_backward(256, 0, 8, 8, 256, 0, 1, 1, 1, 1, 8, 1.0, top, stats, ids, None, gs, None, 1, a, 1, out, None)
    assert back(stats=None) == back(out=None) == back(top=1, ids=None, a=256) == -4 and back(out=258) == back(stats=8) == -6 and back(gs=2) == -7
