"""Log probabilities, entropies, alternatives and their gradients against the
same formulas in 64 bits.

Tolerances.  Everything is formed from the logits as stored, in fp32: with
u = 2^-24, the sum S of V terms e^(x - m) is off by a relative (log2(V) + 4) u
at most through its tree of additions, plus the hardware exponential's 2 u and
its argument's u (m - x) log2(e) (terms far below the maximum weigh e^(x - m)
of that, at most u / e each relative to the largest).  So ls = log S is off by
about (log2(V) + 8) u < 28 u = 1.7e-6 absolutely, and log p by that plus its own
two roundings of u |log p|.  H = ls - T / S is off by twice that relative to
its terms, |T| / S <= log V.  p is off by (28 + |log p| log2(e) + 3) u
relative.  An output of 16 bits adds its half step.
"""
import math

import pytest
import torch

import lite_ssm_amd as L

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ACT = {"f16": (L.F16, torch.float16), "bf16": (L.BF16, torch.bfloat16), "f32": (L.F32, torch.float32)}


def exact(x, tokens, k):
    """(logprob, entropy, (m, ls), top ids, top log p) in 64 bits, by the rules
    of the header."""
    x = x.double().cpu()
    M, V = x.shape
    m = x.max(-1).values
    empty = m == -math.inf
    m = torch.where(empty, 0.0, m)
    e = torch.exp(x - m[:, None])
    S = e.sum(-1)
    ls = torch.where(empty, math.inf, torch.log(S))
    lp = (x - m[:, None]) - ls[:, None]
    p = torch.exp(lp)
    H = -torch.where(p > 0, p * lp, 0.0).sum(-1)
    H = torch.where(torch.isnan(S), math.nan, H)
    t = tokens.cpu().long()
    given = torch.where(t < 0, 0.0, lp.gather(1, t.clamp(0, V - 1)[:, None])[:, 0])
    ids, best = torch.full((M, k), -1), torch.full((M, k), -math.inf, dtype=torch.float64)
    for r in range(M if k else 0):
        row = x[r].tolist()
        order = sorted((i for i in range(V) if row[i] > -math.inf), key=lambda i: (-row[i], i))[:k]
        for j, i in enumerate(order):
            ids[r, j], best[r, j] = i, lp[r, i]
    return given, H, torch.stack([m, ls], -1), ids, best, lp, p


def call(ctx, x, tokens, k, act, stride=0, ws=True):
    M, V = tokens.shape[0], x.shape[1]
    kw = dict(device="cuda")
    o = dict(logprob=torch.full((M,), 7.0, **kw), entropy=torch.full((M,), 7.0, **kw), stats=torch.full((M, 2), 7.0, **kw),
             top_ids=torch.full((M, k), 7, dtype=torch.int32, **kw), top_logprobs=torch.full((M, k), 7.0, **kw))
    n = ctx.token_logprobs_workspace(M, V, k)
    w = torch.full((n,), 0x5a, dtype=torch.uint8, **kw) if n else None
    ctx.token_logprobs(x, tokens, o["logprob"], o["entropy"], o["stats"], o["top_ids"], o["top_logprobs"], M, V, k, act,
                       w, stride)
    torch.cuda.synchronize()
    return {n: v.cpu() for n, v in o.items()}


def close(got, want, bound, what):
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]) and torch.equal(torch.isinf(got), inf), what
    fine = torch.isfinite(want)
    d = (got - want).abs()[fine]
    b = bound[fine] if isinstance(bound, torch.Tensor) else torch.full_like(d, bound)
    assert bool((d <= b).all()), f"{what}: {float((d / b).max()):.3g} of the bound"


def check(ctx, x, tokens, k, act):
    got = call(ctx, x, tokens, k, act)
    lp, H, stats, ids, best, _, _ = exact(x, tokens, k)
    V = x.shape[1]
    ls_err = 28 * U
    close(got["logprob"], lp, ls_err + 2 * U * lp.abs().nan_to_num(0, 0, 0), "logprob")
    close(got["entropy"], H, 3 * ls_err * (1 + math.log(V)), "entropy")
    close(got["stats"][:, 0], stats[:, 0], 0.0, "max")
    close(got["stats"][:, 1], stats[:, 1], ls_err + U * stats[:, 1].abs().nan_to_num(0, 0, 0), "log sum")
    if k:
        assert torch.equal(got["top_ids"].long(), ids), "alternatives"
        close(got["top_logprobs"], best, ls_err + 2 * U * best.abs().nan_to_num(0, 0, 0), "their log p")


def logits(M, V, dt, seed, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, V, generator=g) * scale).to(dt)
    t = torch.randint(0, V, (M,), generator=g, dtype=torch.int32)
    return x.cuda(), t.cuda()


# vocabularies of one element, of ragged ends, of one and of several segments
# (8192 vectors: 65536 values of 16 bits, 32768 of 32)
@pytest.mark.parametrize("act", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("V,k", [(1, 1), (2, 2), (7, 3), (63, 5), (1000, 20), (8191, 64), (16385, 4), (32769, 20),
                                 (65541, 20), (131073, 7)])
def test_rows(ctx, act, V, k):
    code, dt = ACT[act]
    x, t = logits(3, V, dt, V + k)
    t[1] = -1
    check(ctx, x, t, k, code)


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("V", [37, 50281, 70000])
def test_masked_and_special_rows(ctx, act, V):
    """Rows of -inf, of the type's lowest value, one value left, equal values
    (ties), NaN, +inf, zeros of both signs, and far apart values."""
    code, dt = ACT[act]
    x, t = logits(10, V, dt, V)
    x[0] = -math.inf
    x[1] = torch.finfo(dt).min
    x[2] = -math.inf
    x[2, V // 2] = -3.0
    t[2] = V // 2
    x[3] = 1.5                                       # all equal: the first ids
    x[4, 5] = math.nan
    x[5, 5] = math.inf
    x[6, ::2], x[6, 1::2] = 0.0, -0.0
    x[7] = torch.finfo(dt).min
    x[7, V - 1] = 4.0                                # the lowest value as a mask
    x[8] = -math.inf
    x[8, 3], x[8, 7], x[8, V - 1] = 1.0, 2.0, 2.0    # fewer left than asked for
    t[8] = 0                                         # a masked token
    x[9, 0], x[9, 1] = torch.finfo(dt).max, torch.finfo(dt).min
    check(ctx, x, t, 6, code)


@pytest.mark.parametrize("act,offset,stride", [("bf16", 0, 1003), ("bf16", 3, 1001), ("f16", 1, 66000), ("f32", 1, 1000),
                                               ("f32", 3, 40003)])
def test_strides_and_unaligned_rows(ctx, act, offset, stride):
    code, dt = ACT[act]
    M, V = 5, stride - 1
    g = torch.Generator().manual_seed(3)
    buf = torch.full((offset + M * stride,), 99.0).to(dt)
    view = buf[offset:].reshape(M, stride)
    view[:, :V] = (torch.randn(M, V, generator=g) * 3).to(dt)
    t = torch.randint(0, V, (M,), generator=g, dtype=torch.int32).cuda()
    x = buf.cuda()[offset:].reshape(M, stride)[:, :V]
    k = 5
    got = call(ctx, x, t, k, code, stride=stride)
    lp, H, stats, ids, best, _, _ = exact(x, t, k)
    close(got["logprob"], lp, 28 * U + 2 * U * lp.abs(), "logprob")
    assert torch.equal(got["top_ids"].long(), ids)


def grads(x, t, g, ge):
    lp, p = exact(x, t, 0)[5:]
    H = exact(x, t, 0)[1]
    V = x.shape[1]
    t = t.cpu().long()
    hot = torch.zeros_like(p)
    on = (t >= 0) & ~torch.isinf(exact(x, t, 0)[2][:, 1])
    hot[torch.arange(len(t))[on], t[on]] = 1.0
    g = torch.where(t >= 0, g.double().cpu(), 0.0)
    plog = torch.where(p > 0, p * (lp + H[:, None]), 0.0)
    d = g[:, None] * (hot - p) - ge.double().cpu()[:, None] * plog
    nan = torch.isnan(p).any(-1)
    d[nan] = math.nan
    # relative error of p (see above) times what it multiplies, and of H
    rel = (31 + 1.45 * lp.abs().clamp(max=150).nan_to_num(150)) * U
    err = rel * p * (g.abs()[:, None] + ge.double().cpu().abs()[:, None] * (lp + H[:, None]).abs().clamp(max=200).nan_to_num(0))
    err = err + p * ge.double().cpu().abs()[:, None] * 84 * U * (1 + math.log(V)) + 4 * U * d.abs().nan_to_num(0)
    return d, err


@pytest.mark.parametrize("act", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("V", [1, 9, 1000, 32773, 50280, 70001])
@pytest.mark.parametrize("how", ["bwd", "grad", "in place"])
def test_gradient(ctx, act, V, how):
    code, dt = ACT[act]
    M = 4
    x, t = logits(M, V, dt, V + 1)
    t[2] = -1
    x[3, V // 2:] = -math.inf
    if V > 1:
        t[3] = 0
    gen = torch.Generator().manual_seed(5)
    g, ge = torch.randn(M, generator=gen).cuda(), torch.randn(M, generator=gen).cuda()
    if V == 1:
        x[3] = 1.0
    want, err = grads(x, t, g, ge)
    kw = dict(device="cuda")
    lp, H, st = torch.empty(M, **kw), torch.empty(M, **kw), torch.empty(M, 2, **kw)
    n = ctx.token_logprobs_workspace(M, V, 0)
    ws = torch.empty(n, dtype=torch.uint8, **kw) if n else None
    inp = x.clone()
    d = inp if how == "in place" else torch.full_like(x, 7.0)
    if how == "bwd":
        ctx.token_logprobs(inp, t, lp, H, st, None, None, M, V, 0, code, ws)
        ctx.token_logprobs_bwd(inp, t, st, H, g, ge, d, M, V, code)
    else:
        ctx.token_logprobs_grad(inp, t, g, ge, lp, H, st, d, M, V, code, ws)
    torch.cuda.synchronize()
    bound = err + (torch.finfo(dt).eps / 2 * want.abs() + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps)
    close(d.cpu(), want, bound, "gradient")
    close(lp.cpu(), exact(x, t, 0)[0], 28 * U + 2 * U * exact(x, t, 0)[0].abs(), "logprob")


@pytest.mark.parametrize("V", [50, 70000])
def test_gradient_of_masked_rows(ctx, V):
    """Nothing left: a zero gradient; NaN: a NaN row, its neighbours untouched."""
    x, t = logits(4, V, torch.bfloat16, 9)
    x[0] = -math.inf
    x[1] = torch.finfo(torch.bfloat16).min
    x[2, 3] = math.nan
    g, ge = torch.ones(4, device="cuda"), torch.ones(4, device="cuda")
    want, err = grads(x, t, g, ge)
    want[0] = 0.0
    lp, H, st = (torch.empty(4, device="cuda"), torch.empty(4, device="cuda"), torch.empty(4, 2, device="cuda"))
    n = ctx.token_logprobs_workspace(4, V, 0)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda") if n else None
    d1, d2 = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    ctx.token_logprobs_grad(x, t, g, ge, lp, H, st, d1, 4, V, L.BF16, ws)
    ctx.token_logprobs_bwd(x, t, st, H, g, ge, d2, 4, V, L.BF16)
    for d in (d1, d2):
        close(d.cpu(), want, err + 2.0 ** -8 * want.abs(), "gradient")
        assert not bool(d[0].any())


def test_gradient_against_differences(ctx):
    """d_logits of a weighted sum of log probabilities and entropies against
    central differences of the forward entry itself.  Step h = 2^-5: the forward
    values are off by 28 u, their difference over 2 h by 28 u / h = 5.4e-5; the
    third derivatives are below 2, their share h^2 / 6 * 2 = 3.3e-4."""
    M, V, h = 2, 12, 2.0 ** -5
    x, t = logits(M, V, torch.float32, 4, scale=1.0)
    g, ge = torch.tensor([0.7, -0.4], device="cuda"), torch.tensor([0.3, 0.9], device="cuda")
    lp, H, st, d = (torch.empty(M, device="cuda"), torch.empty(M, device="cuda"), torch.empty(M, 2, device="cuda"),
                    torch.empty_like(x))
    ctx.token_logprobs_grad(x, t, g, ge, lp, H, st, d, M, V, L.F32)

    def loss(y):
        o = call(ctx, y, t, 0, L.F32)
        return g.cpu().double() * o["logprob"].double() + ge.cpu().double() * o["entropy"].double()
    for v in range(V):
        e = torch.zeros_like(x)
        e[:, v] = h
        num = (loss(x + e) - loss(x - e)) / (2 * h)
        assert bool(((num - d[:, v].cpu().double()).abs() < 6e-4).all()), v


def test_optional_outputs_and_no_rows(ctx):
    x, t = logits(2, 100, torch.float32, 1)
    H = torch.full((2,), 7.0, device="cuda")
    ctx.token_logprobs(x, None, None, H, None, None, None, 2, 100, 0, L.F32)
    assert bool((H < 5).all())
    ctx.token_logprobs(None, None, None, None, None, None, None, 0, 100, 0, L.F32)
    d = torch.full_like(x, 7.0)
    st = torch.zeros(2, 2, device="cuda")
    ctx.token_logprobs(x, t, None, None, st, None, None, 2, 100, 0, L.F32)
    ctx.token_logprobs_bwd(x, None, st, None, None, None, d, 2, 100, L.F32)
    assert not bool(d.any())          # no upstream gradient


def test_a_token_beyond_the_vocabulary_is_reported(ctx):
    x, t = logits(3, 100, torch.float32, 1)
    t[1] = 100
    lp = torch.zeros(3, device="cuda")
    with pytest.raises(L.LssmError, match="not below the vocabulary") as e:
        ctx.token_logprobs(x, t, lp, None, None, None, None, 3, 100, 0, L.F32)
    assert e.value.code == 1
    assert torch.isnan(lp).tolist() == [False, True, False]
    ctx.sync()                        # reported once


def test_many_rows_with_other_rows_left_alone(ctx):
    """More rows than blocks run at once; what lies behind the last row stays."""
    M, V, pad = 1500, 333, 5
    x, t = logits(M, V, torch.bfloat16, 8)
    lp, H = torch.full((M + pad,), 7.0, device="cuda"), torch.full((M + pad,), 7.0, device="cuda")
    d = torch.full((M + pad, V), 7.0, dtype=torch.bfloat16, device="cuda")
    st = torch.full((M + pad, 2), 7.0, device="cuda")
    g = torch.ones(M, device="cuda")
    ctx.token_logprobs_grad(x, t, g, None, lp, H, st, d, M, V, L.BF16)
    want = torch.log_softmax(x.double(), -1)
    assert bool(((lp[:M] - want[torch.arange(M, device="cuda"), t.long()]).abs() < 4e-6).all())
    for v in (lp, H, d, st):
        assert bool((v[M:] == 7.0).all())


@pytest.mark.parametrize("V,k", [(50280, 5), (131072, 20)])
def test_captured_and_replayed(ctx, V, k):
    """A captured call and its gradient give the eager results on every replay,
    with eager work of the same context between them."""
    M = 3
    x, t = logits(M, V, torch.bfloat16, 2)
    y, _ = logits(M, V, torch.bfloat16, 12)
    kw = dict(device="cuda")
    lp, H, st = torch.empty(M, **kw), torch.empty(M, **kw), torch.empty(M, 2, **kw)
    ids, tl = torch.empty(M, k, dtype=torch.int32, **kw), torch.empty(M, k, **kw)
    n = ctx.token_logprobs_workspace(M, V, k)
    ws = torch.empty(n, dtype=torch.uint8, **kw) if n else None
    g, d = torch.randn(M, **kw), torch.empty_like(x)
    stream = torch.cuda.ExternalStream(ctx.stream)

    def both():
        ctx.token_logprobs(x, t, lp, H, st, ids, tl, M, V, k, L.BF16, ws)
        ctx.token_logprobs_bwd(x, t, st, H, g, g, d, M, V, L.BF16)
    ctx.begin_batch()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        both()
    ctx.commit_and_wait()
    keep = x.clone()
    for i in range(4):
        x.copy_(keep if i % 2 else y)
        both()
        torch.cuda.synchronize()
        want = [v.clone() for v in (lp, H, st, ids, tl, d)]
        for v in (lp, H, st, tl, d):
            v.fill_(3.0)
        ids.fill_(3)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((lp, H, st, ids, tl, d), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("V", [50280, 131072])
def test_equal_logits_have_equal_log_probabilities(ctx, V):
    """Many ties among the likeliest of many rows: equal logits get the same
    bits, in the order of their ids, and a second call gives the same bits."""
    M, k = 600, 20
    x, t = logits(M, V, torch.bfloat16, 3)
    x = (x * 4).round() / 4
    code = L.BF16
    a, b = call(ctx, x, t, k, code), call(ctx, x, t, k, code)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    v = x.cpu().gather(1, a["top_ids"].long())
    lp = a["top_logprobs"]
    same = v[:, 1:] == v[:, :-1]
    assert bool(same.any())
    assert torch.equal(lp[:, 1:] == lp[:, :-1], same)
    assert bool((a["top_ids"][:, 1:] > a["top_ids"][:, :-1])[same].all())


@pytest.mark.parametrize("M", [1, 5, 40])
@pytest.mark.parametrize("V", [4097, 50281, 140000])
@pytest.mark.parametrize("how", ["ascending", "descending", "one value", "one wave", "alternating"])
def test_alternatives_of_uneven_rows(ctx, M, V, how):
    """Where the best logits lie together, or are all alike, and as many
    alternatives as a row gives."""
    i = torch.arange(V, device="cuda", dtype=torch.float32)
    x = {"ascending": i / V, "descending": -i / V, "one value": 0 * i + 1,
         "one wave": torch.where((i >= 512) & (i < 600), 5 + (i % 7), -i / V),
         "alternating": torch.where(i % 2 == 0, 1.0, -1.0)}[how].repeat(M, 1)
    t = torch.arange(M, dtype=torch.int32, device="cuda")
    got = call(ctx, x, t, 64, L.F32)
    ids = torch.sort(x[0].cpu(), descending=True, stable=True).indices[:64].int()
    assert all(torch.equal(got["top_ids"][r], ids) for r in range(M))
    lp = torch.log_softmax(x[0].double(), -1).cpu()[ids.long()]
    bound = 28 * U + 2 * U * lp.abs()
    for r in range(M):
        close(got["top_logprobs"][r], lp, bound, "top_logprobs")


@pytest.mark.parametrize("V,k", [(50280, 20), (256000, 5)])
def test_a_workspace_for_many_rows_serves_fewer(ctx, V, k):
    x, t = logits(40, V, torch.bfloat16, 5)
    ws = torch.empty(ctx.token_logprobs_workspace(40, V, k), dtype=torch.uint8, device="cuda")
    for M in (40, 31, 4, 1):
        lp, ids = torch.empty(M, device="cuda"), torch.empty(M, k, dtype=torch.int32, device="cuda")
        ctx.token_logprobs(x[:M], t[:M], lp, None, None, ids, torch.empty(M, k, device="cuda"), M, V, k, L.BF16, ws)
        want = exact(x[:M], t[:M], k)
        close(lp.cpu(), want[0], 28 * U + 2 * U * want[0].abs(), "logprob")
        assert torch.equal(ids.cpu().long(), want[3])


def test_gradient_rows_between_the_logits_rows(ctx):
    """Rows of logits and of their gradient that take turns in one array."""
    M, V = 5, 1000
    x, t = logits(M, V, torch.float16, 9)
    both = torch.full((M, 2, V), 3.0, dtype=torch.float16, device="cuda")
    both[:, 0] = x
    g = torch.ones(M, device="cuda")
    st, H, want = torch.empty(M, 2, device="cuda"), torch.empty(M, device="cuda"), torch.empty_like(x)
    ctx.token_logprobs_grad(x, t, g, None, None, H, st, want, M, V, L.F16)
    ctx.token_logprobs_grad(both, t, g, None, None, H, st, both[0, 1], M, V, L.F16, stride=2 * V, d_stride=2 * V)
    assert torch.equal(both[:, 0], x) and torch.equal(both[:, 1], want)
