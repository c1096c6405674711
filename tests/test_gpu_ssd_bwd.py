"""The scan's gradients against the recurrences in 64 bits.

Tolerances.  Every result is a sum; with u = 2^-24 a sum of n fp32 terms is off
by at most n u times the sum of the terms' absolute values, which
ssd_bwd_ref.grads(absolute=True) gives.  The longest chain of additions behind a
result: N or P terms of a product (256), the tokens of a chunk (64), the
chunks' carries (whose decays shrink them: 8), the group's heads (16 here), and
about 50 roundings of factors (softplus, exponentials, decays, scalings): under
400 u.  With 16-bit inputs an operand formed in fp32 may be taken as a pair of
bf16 numbers, 2^-17 each, two such operands at most: 400 u + 2^-16.  To that
comes half a step of the output's type.
"""
import pytest
import torch

import lite_ssm_amd as L
from ssd_bwd_ref import NAMES, grads

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ACT = {"f16": (L.F16, torch.float16), "bf16": (L.BF16, torch.bfloat16), "f32": (L.F32, torch.float32)}


def inputs(dt, b, n, H, P, G, N, seed, state=True, dt_scale=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    v = dict(X=r(b, n, H, P), B=r(b, n, G, N) / N ** 0.5, C=r(b, n, G, N) / N ** 0.5, dt=dt_scale * r(b, n, H),
             dt_bias=r(H) - 2, A_log=torch.log(1 + 15 * torch.rand(H, generator=g)), D=r(H), dY=r(b, n, H, P))
    v = {k: t.to(dt) for k, t in v.items()}
    for k in ("state", "d_state"):
        v[k] = r(b, H, P, N) if state else torch.zeros(b, H, P, N)
    return v


def outputs(v):
    o = {"d" + k if k not in ("dt", "dt_bias") else "d_" + k: torch.full_like(v[k], 7.0, device="cuda")
         for k in ("X", "B", "C", "dt", "dt_bias", "A_log", "D")}
    return dict(o, d_state0=torch.full_like(v["state"], 7.0, device="cuda"))


def dims(v, lo=1e-6, hi=1e6, has_D=1):
    b, n, H, P = v["X"].shape
    G, N = v["B"].shape[2:]
    return L.SSDDims(n, H, P, N, G, 64, lo, hi, has_D)


def workspace(ctx, v, d, act, tail=256):
    """Exactly the bytes asked for, in front of a stretch that has to stay as it is."""
    n = ctx.ssd_chunked_bwd_workspace(v["X"].shape[0], d, act)
    buf = torch.full((n + tail,), 0xff, dtype=torch.uint8, device="cuda")     # NaN wherever it is read unwritten
    return buf, buf[:n]


def call(ctx, v, act, state=True, lo=1e-6, hi=1e6, has_D=1):
    t = {k: x.cuda() for k, x in v.items()}
    o, d = outputs(v), dims(v, lo, hi, has_D)
    buf, ws = workspace(ctx, v, d, act)
    ctx.ssd_chunked_bwd(t["X"], t["B"], t["C"], t["dt"], t["dt_bias"], t["A_log"], t["D"] if has_D else None,
                        t["state"] if state else None, t["dY"], t["d_state"] if state else None, o["dX"], o["dB"], o["dC"],
                        o["d_dt"], o["d_dt_bias"], o["dA_log"], o["dD"] if has_D else None, o["d_state0"],
                        v["X"].shape[0], d, act, ws)
    torch.cuda.synchronize()
    assert bool((buf[len(ws):] == 0xff).all()), "the workspace was left"
    return {k: x.cpu() for k, x in o.items()}


def check(got, v, dt, lo=1e-6, hi=1e6, skip=()):
    want, mag = grads(v, lo, hi), grads(v, lo, hi, absolute=True)
    rel = 400 * U + (0 if dt is torch.float32 else 2.0 ** -16)
    for k in NAMES:
        if k in skip:
            continue
        half = 0.0 if got[k].dtype is torch.float32 else torch.finfo(dt).eps / 2
        bound = rel * (1 + half) * mag[k] + half * want[k].abs() + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
        d = (got[k].double() - want[k]).abs()
        assert bool((d <= bound).all()), f"{k}: {float((d / bound).max()):.3g} of the bound"


# lengths around the chunks' ends
@pytest.mark.parametrize("act", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257])
def test_lengths(ctx, act, n):
    code, dt = ACT[act]
    v = inputs(dt, 2, n, 4, 64, 2, 128, n)
    check(call(ctx, v, code), v, dt)


# head and state sizes inside, at and past the tiles
@pytest.mark.parametrize("act", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,P,G,N", [(1, 1, 1, 1), (2, 8, 1, 16), (3, 33, 3, 63), (4, 32, 1, 64), (6, 80, 2, 65),
                                     (2, 128, 2, 128), (2, 64, 1, 200), (5, 20, 1, 256), (2, 130, 1, 129), (16, 64, 1, 128)])
def test_sizes(ctx, act, H, P, G, N):
    code, dt = ACT[act]
    v = inputs(dt, 1, 70, H, P, G, N, H + P + N)
    check(call(ctx, v, code), v, dt)


# several chunks, slices and groups at once, head counts around those that share
# an XCD or a block
@pytest.mark.parametrize("act", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("b,n,H,P,G,N", [(2, 400, 12, 64, 3, 128), (1, 700, 5, 128, 1, 128), (3, 130, 9, 192, 9, 128),
                                         (2, 333, 7, 40, 7, 100), (1, 513, 24, 64, 1, 64)])
def test_many_chunks_slices_and_groups(ctx, act, b, n, H, P, G, N):
    code, dt = ACT[act]
    v = inputs(dt, b, n, H, P, G, N, 17 * n + H)
    check(call(ctx, v, code), v, dt)


@pytest.mark.parametrize("act", ["f32", "bf16", "f16"])
def test_no_states_no_D(ctx, act):
    code, dt = ACT[act]
    v = inputs(dt, 1, 100, 4, 64, 1, 128, 5, state=False)
    v["D"] = torch.zeros_like(v["D"])
    got = call(ctx, v, code, state=False, has_D=0)
    check(got, v, dt, skip=("dD",))
    assert bool((got["dD"] == 7.0).all())


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("dt_scale", [0.0, 3.0, 12.0])
def test_slow_fast_and_clamped_steps(ctx, act, dt_scale):
    """Step sizes from e^-30 to 30: decays that underflow within a chunk, and
    both ends of the clamp (the values that meet it have no gradient)."""
    code, dt = ACT[act]
    v = inputs(dt, 1, 150, 4, 64, 1, 128, 11, dt_scale=dt_scale)
    check(call(ctx, v, code, lo=1e-3, hi=5.0), v, dt, lo=1e-3, hi=5.0)


@pytest.mark.parametrize("act", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("big", [30.0, 1000.0])
def test_steps_that_forget_everything(ctx, act, big):
    """Some steps as large as softplus gives them (no upper clamp), ordinary ones
    behind them: a chunk's sums of A dt pass 10^5, and the decays of the ordinary
    steps are as exact as before."""
    code, dt = ACT[act]
    v = inputs(dt, 2, 300, 4, 64, 2, 128, 41)
    g = torch.Generator().manual_seed(42)
    v["dt"] = torch.where(torch.rand(2, 300, 4, generator=g) < 0.3, torch.tensor(big, dtype=dt), v["dt"])
    check(call(ctx, v, code, lo=0.0, hi=float("inf")), v, dt, lo=0.0, hi=float("inf"))


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_a_head_that_is_nan(ctx, act):
    """Its gradients are NaN, and its group's dB and dC; the other group's are not touched."""
    code, dt = ACT[act]
    v = inputs(dt, 1, 200, 4, 64, 2, 128, 43)
    v["A_log"][1] = float("nan")
    got = call(ctx, v, code)
    assert bool(got["dX"][:, :-1, 1].isnan().all()) and bool(got["dC"][:, 1:, 0].isnan().all())
    assert bool(got["dB"][:, :-1, 0].isnan().all()) and bool(got["d_state0"][:, 1].isnan().all())
    for k in ("dX", "d_dt"):
        got[k][:, :, 1] = 0
    for k in ("dB", "dC"):
        got[k][:, :, 0] = 0
    for k in ("d_dt_bias", "dA_log", "dD"):
        got[k][1] = 0
    got["d_state0"][:, 1] = 0
    assert all(bool(x.isfinite().all()) for x in got.values())
    v["A_log"][1] = 0
    want = call(ctx, v, code)
    assert torch.equal(got["dX"][:, :, 2:], want["dX"][:, :, 2:]) and torch.equal(got["dB"][:, :, 1], want["dB"][:, :, 1])


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_nothing_to_scan(ctx, act):
    """No tokens: the state's gradient passes through, parameters have none.
    No sequences: the parameters' gradients are written all the same."""
    code, dt = ACT[act]
    v = inputs(dt, 2, 0, 4, 64, 1, 128, 3)
    got = call(ctx, v, code)
    assert torch.equal(got["d_state0"], v["d_state"])
    for k in ("d_dt_bias", "dA_log", "dD"):
        assert not bool(got[k].any())
    got = call(ctx, inputs(dt, 0, 9, 4, 64, 1, 128, 3), code)
    for k in ("d_dt_bias", "dA_log", "dD"):
        assert not bool(got[k].any())


@pytest.mark.parametrize("act", ["f32", "bf16", "f16"])
def test_unaligned_arrays(ctx, act):
    """Arrays one element off a 16-byte address."""
    code, dt = ACT[act]
    v = inputs(dt, 1, 77, 2, 64, 1, 128, 21)
    t = {}
    for k, x in v.items():
        buf = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
        t[k] = buf[1:].view(x.shape).copy_(x)
    o = {}
    for k, x in outputs(v).items():
        buf = torch.full((x.numel() + 2,), 7.0, dtype=x.dtype, device="cuda")
        o[k] = (buf, buf[1:-1].view(x.shape))
    d = dims(v)
    buf, ws = workspace(ctx, v, d, code)
    p = {k: x[1] for k, x in o.items()}
    ctx.ssd_chunked_bwd(t["X"], t["B"], t["C"], t["dt"], t["dt_bias"], t["A_log"], t["D"], t["state"], t["dY"], t["d_state"],
                        p["dX"], p["dB"], p["dC"], p["d_dt"], p["d_dt_bias"], p["dA_log"], p["dD"], p["d_state0"], 1, d, code,
                        ws)
    torch.cuda.synchronize()
    check({k: x.cpu() for k, x in p.items()}, v, dt)
    for k, (b, _) in o.items():
        assert float(b[0]) == 7.0 and float(b[-1]) == 7.0, k


@pytest.mark.parametrize("act", ["f32", "bf16", "f16"])
def test_same_bits_twice_and_replayed(ctx, act):
    """The same inputs give the same bits: eagerly, captured and on every replay,
    with other work of the context and new inputs between them."""
    code, dt = ACT[act]
    v, other = (inputs(dt, 2, 300, 4, 64, 2, 128, s) for s in (1, 2))
    t = {k: x.cuda() for k, x in v.items()}
    o, d = outputs(v), dims(v)
    ws = workspace(ctx, v, d, code)[1]
    names = ("dX", "dB", "dC", "d_dt", "d_dt_bias", "dA_log", "dD", "d_state0")

    def run():
        ctx.ssd_chunked_bwd(t["X"], t["B"], t["C"], t["dt"], t["dt_bias"], t["A_log"], t["D"], t["state"], t["dY"],
                            t["d_state"], *(o[k] for k in names), 2, d, code, ws)
    stream = torch.cuda.ExternalStream(ctx.stream)
    ctx.begin_batch()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run()
    ctx.commit_and_wait()
    for i in range(4):
        for k, x in (other if i % 2 else v).items():
            t[k].copy_(x)
        run()
        torch.cuda.synchronize()
        want = {k: o[k].clone() for k in names}
        for k in names:
            o[k].fill_(3.0)
        ws.fill_(0xff)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k in names:
            assert torch.equal(o[k], want[k]), k
        if i == 0:
            check({k: x.cpu() for k, x in want.items()}, v, dt)


def test_against_differences(ctx):
    """A directional derivative of the forward entry (fp32) in X, B, C, dt and
    state against the gradients' inner product.  The forward's sums are off by
    about 1e-6 of their size 30 a step of 2^-7 in a unit direction: 4e-3; the third
    derivative's share is of that order too."""
    b, n, H, P, G, N = 1, 20, 2, 64, 1, 128
    v = inputs(torch.float32, b, n, H, P, G, N, 31)
    got = call(ctx, v, L.F32)
    g = torch.Generator().manual_seed(2)
    way = {k: torch.randn(v[k].shape, generator=g) for k in ("X", "B", "C", "dt", "state")}
    size = sum(float(x.square().sum()) for x in way.values()) ** 0.5
    way = {k: x / size for k, x in way.items()}

    def loss(h):
        t = {k: (x + h * way[k] if k in way else x).cuda() for k, x in v.items()}
        y, st = torch.empty_like(t["X"]), t["state"].clone()
        ctx.ssd_chunked(t["X"], t["B"], t["C"], t["dt"], t["dt_bias"], t["A_log"], t["D"], y, st, b,
                        L.SSDDims(n, H, P, N, G, 20, 1e-6, 1e6, 1), L.F32)
        torch.cuda.synchronize()
        return float((y.double().cpu() * v["dY"].double()).sum() + (st.double().cpu() * v["d_state"].double()).sum())
    h = 2.0 ** -7
    num = (loss(h) - loss(-h)) / (2 * h)
    names = dict(X="dX", B="dB", C="dC", dt="d_dt", state="d_state0")
    want = sum(float((got[names[k]].double() * way[k].double()).sum()) for k in way)
    assert abs(num - want) < 1e-2 * max(1.0, abs(want)), (num, want)


def test_two_contexts_at_once(ctx):
    """Two streams, a workspace each, calls in turn without waiting."""
    cases = [("bf16", inputs(torch.bfloat16, 1, 500, 8, 64, 1, 128, 51)), ("f32", inputs(torch.float32, 2, 200, 4, 64, 2, 128, 52))]
    want = [call(ctx, v, ACT[a][0]) for a, v in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    ctxs = [L.Ctx(stream=s.cuda_stream) for s in streams]
    runs = []
    for c, (a, v) in zip(ctxs, cases):
        t, o, d = {k: x.cuda() for k, x in v.items()}, outputs(v), dims(v)
        runs.append((c, t, o, d, workspace(c, v, d, ACT[a][0])[1], ACT[a][0], v["X"].shape[0]))
    torch.cuda.synchronize()
    for c in ctxs:
        c.begin_batch()
    for _ in range(20):
        for c, t, o, d, ws, code, b in runs:
            c.ssd_chunked_bwd(t["X"], t["B"], t["C"], t["dt"], t["dt_bias"], t["A_log"], t["D"], t["state"], t["dY"],
                              t["d_state"], o["dX"], o["dB"], o["dC"], o["d_dt"], o["d_dt_bias"], o["dA_log"], o["dD"],
                              o["d_state0"], b, d, code, ws)
    for c in ctxs:
        c.commit_and_wait()
    for (c, t, o, *_), w in zip(runs, want):
        for k in w:
            assert torch.equal(o[k].cpu(), w[k]), k
        c.close()
