"""The scan's gradient on the CPU: the 64-bit recurrences that the kernels are
held to against torch's own differentiation of the forward, and what the entry
refuses (every check comes before the launch, so no GPU is touched)."""
import ctypes as C

import pytest
import torch

import lite_ssm_amd as L
from ssd_bwd_ref import NAMES, forward, grads

CTX = C.addressof(C.create_string_buffer(4096))
P = 1 << 20


@pytest.mark.parametrize("b,n,H,p,G,N", [(2, 7, 4, 3, 2, 5), (1, 1, 2, 2, 1, 4), (1, 12, 3, 4, 3, 2)])
def test_the_recurrences_are_the_forward_s_gradient(b, n, H, p, G, N):
    g = torch.Generator().manual_seed(n)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    v = dict(X=r(b, n, H, p), B=r(b, n, G, N), C=r(b, n, G, N), dt=r(b, n, H), dt_bias=r(H) - 1, A_log=r(H), D=r(H),
             state=r(b, H, p, N))
    dY, d_state = r(b, n, H, p), r(b, H, p, N)
    lo, hi = 0.05, 1.2                     # both ends of the clamp are met
    leaves = {k: t.clone().requires_grad_() for k, t in v.items()}
    y, h = forward(leaves, lo, hi)
    ((y * dY).sum() + (h * d_state).sum()).backward()
    got = grads(dict(v, dY=dY, d_state=d_state), lo, hi)
    for name, leaf in zip(NAMES, ("X", "B", "C", "dt", "dt_bias", "A_log", "D", "state")):
        want = leaves[leaf].grad
        assert torch.allclose(got[name], want, rtol=1e-10, atol=1e-12), name
    mag = grads(dict(v, dY=dY, d_state=d_state), lo, hi, absolute=True)
    for name in NAMES:
        assert bool((mag[name] >= got[name].abs() - 1e-12).all()), name


def call(ctx=CTX, batch=1, dims=None, act=L.BF16, ws=P, n=1 << 40, **over):
    d = dict(L=10, H=4, P=8, N=16, G=2, chunk=8, has_D=1)
    d.update(dims or {})
    names = ["X", "B", "C", "dt", "dt_bias", "A_log", "D", "state", "dY", "d_state", "dX", "dB", "dC", "d_dt", "d_dt_bias",
             "dA_log", "dD", "d_state0"]
    a = {k: P for k in names}
    a.update(over)
    s = L.SSDDims(d["L"], d["H"], d["P"], d["N"], d["G"], d["chunk"], 0.0, 1e6, d["has_D"])
    return L.lib.lssm_ssd_chunked_bwd(ctx, *(a[k] for k in names), batch, s, act, ws, n)


@pytest.mark.parametrize("kw,text", [
    (dict(ctx=None), "null lssm_ctx"),
    (dict(act=9), "unknown dtype"),
    (dict(dims=dict(H=0)), "must be > 0"),
    (dict(dims=dict(G=3)), "multiple of n_groups"),
    (dict(dims=dict(N=257)), "N must be <= 256"),
    (dict(dims=dict(P=1025)), "P must be <= 1024"),
    (dict(dims=dict(L=1048577)), "L <="),
    (dict(batch=65536), "batch must be"),
    (dict(D=None), "has_D set"),
    (dict(dD=None), "has_D set"),
    (dict(X=None), "null pointer"),
    (dict(dY=None), "null pointer"),
    (dict(dA_log=None), "null pointer"),
    (dict(dX=P + 1), "aligned to their type"),
    (dict(B=P + 2, act=L.F32), "aligned to their type"),
    (dict(state=P + 2), "states must be 4-byte"),
    (dict(ws=None), "workspace needs"),
    (dict(n=100), "workspace needs"),
    (dict(ws=P + 8), "16-byte aligned"),
    (dict(dims=dict(L=1048576, H=256, G=256, P=1, N=1)), "too large"),
    (dict(), "overlaps an input"),
])
def test_refuses(kw, text):
    assert call(**kw) == 1
    assert text in L.lib.lssm_last_error().decode()


@pytest.mark.parametrize("where,text", [
    (dict(dX="X"), "overlaps an input"),
    (dict(d_state0="state"), "overlaps an input"),
    (dict(dB="dY"), "overlaps an input"),
    (dict(dA_log="A_log"), "overlaps an input"),
    (dict(dC="dB"), "outputs overlap"),
    (dict(d_dt="ws"), "the workspace"),
])
def test_refuses_what_overlaps(where, text):
    names = ["X", "B", "C", "dt", "dt_bias", "A_log", "D", "state", "dY", "d_state", "dX", "dB", "dC", "d_dt", "d_dt_bias",
             "dA_log", "dD", "d_state0", "ws"]
    at = {k: P + (i << 16) for i, k in enumerate(names)}
    over = dict(at, n=1 << 16)
    for k, other in where.items():
        over[k] = at[other]
    ws = over.pop("ws")
    assert call(ws=ws, **over) == 1
    assert text in L.lib.lssm_last_error().decode()


def test_workspace_size():
    f = L.lib.lssm_ssd_chunked_bwd_workspace
    d = L.SSDDims(100, 4, 64, 128, 1, 64, 0.0, 1e6, 1)
    one, two = f(1, d, L.BF16), f(2, d, L.BF16)
    assert 0 < one < two
    assert f(1, L.SSDDims(100, 4, 64, 257, 1, 64, 0.0, 1e6, 1), L.BF16) == 0
    big = f(4, L.SSDDims(4096, 80, 64, 128, 1, 64, 0.0, 1e6, 1), L.BF16)
    assert big < 1 << 33
