"""What the log-probability entries refuse, and the sizes of their workspaces: no
GPU is touched, as every check comes before the launch.  The handle is a zeroed
block in place of a context, which a refused call does not look into."""
import ctypes as C

import pytest

import lite_ssm_amd as L

CTX = C.addressof(C.create_string_buffer(4096))
P = 1 << 20          # an aligned address that is never used


def refused(rc, text):
    assert rc == 1, rc
    assert text in L.lib.lssm_last_error().decode()


def fwd(logits=P, stride=0, tokens=P, lp=P, H=P, st=P, ids=None, tl=None, rows=4, V=100, k=0, act=L.BF16, ws=None, n=0,
        ctx=CTX):
    return L.lib.lssm_token_logprobs(ctx, logits, stride, tokens, lp, H, st, ids, tl, rows, V, k, act, ws, n)


@pytest.mark.parametrize("kw,text", [
    (dict(ctx=None), "null lssm_ctx"),
    (dict(act=9), "unknown dtype"),
    (dict(logits=None), "null logits"),
    (dict(V=0), "vocab must be"),
    (dict(V=2097153), "vocab must be"),
    (dict(rows=1 << 24), "rows must be"),
    (dict(rows=1 << 21), "rows must be"),
    (dict(rows=1 << 20, V=32769), "rows must be"),
    (dict(stride=99), "row stride"),
    (dict(logits=P + 1), "not aligned"),
    (dict(logits=P + 2, act=L.F32), "not aligned"),
    (dict(tokens=None), "need tokens"),
    (dict(tokens=P + 2), "4-byte aligned"),
    (dict(st=P + 2), "4-byte aligned"),
    (dict(k=65), "top_k must be"),
    (dict(k=101), "top_k must be"),
    (dict(V=3, k=4, ids=P, tl=P), "top_k must be"),
    (dict(k=1, ids=P), "top_k without"),
    (dict(k=1, tl=P), "top_k without"),
    (dict(V=256000), "workspace needs"),
    (dict(V=256000, ws=P, n=10), "workspace needs"),
    (dict(V=256000, ws=P + 4, n=1 << 30), "8-byte aligned"),
])
def test_forward_refuses(kw, text):
    refused(fwd(**kw), text)


@pytest.mark.parametrize("over,text", [
    (dict(d=None), "null d_logits"),
    (dict(st=None), "null d_logits or stats"),
    (dict(H=None), "needs the entropies"),
    (dict(tokens=None), "need tokens"),
    (dict(d_stride=99), "row stride"),
    (dict(d=P, logits=P, d_stride=104), "equal strides"),
    (dict(d=2 * P + 1), "not aligned"),
    (dict(d=P + 2), "overlaps logits"),
    (dict(d=P + 200), "overlaps logits"),
    (dict(d=P - 798), "overlaps logits"),
    (dict(stride=250, d_stride=250, d=P + 198), "overlaps logits"),
    (dict(stride=250, d_stride=250, d=P + 302), "overlaps logits"),
    (dict(stride=250, d_stride=249, d=P + 200), "overlaps logits"),
])
def test_backward_refuses(over, text):
    a = dict(logits=P, stride=0, tokens=P, st=P, H=P, g=P, ge=P, d=2 * P, d_stride=0)
    a.update(over)
    refused(L.lib.lssm_token_logprobs_bwd(CTX, a["logits"], a["stride"], a["tokens"], a["st"], a["H"], a["g"], a["ge"],
                                          a["d"], a["d_stride"], 4, 100, L.F16), text)


@pytest.mark.parametrize("over,text", [
    (dict(d=None), "null d_logits"),
    (dict(H=None), "stats or entropy"),
    (dict(st=None), "stats or entropy"),
    (dict(V=256000), "workspace needs"),
])
def test_one_pass_refuses(over, text):
    a = dict(logits=P, tokens=P, st=P, H=P, g=P, d=2 * P, V=100)
    a.update(over)
    refused(L.lib.lssm_token_logprobs_grad(CTX, a["logits"], 0, a["tokens"], a["g"], None, None, a["H"], a["st"], a["d"],
                                           0, 4, a["V"], L.F16, None, 0), text)


def test_no_rows_is_nothing_to_do():
    assert fwd(rows=0, logits=None) == 0


def test_workspace_grows_with_what_it_holds():
    f = L.lib.lssm_token_logprobs_workspace
    assert f(8, 100, 5) == 0 and f(800, 2048, 64) == 0
    one, more = f(1, 256000, 0), f(1, 256000, 20)
    assert 0 < one < more
    assert f(1, 2097153, 0) == 0 and f(1, 100, 65) == 0


@pytest.mark.parametrize("k", [0, 5, 64])
@pytest.mark.parametrize("V", [100, 2049, 50280, 65544, 256000, 2097152])
def test_workspace_of_some_rows_is_enough_for_fewer(V, k):
    sizes = [L.lib.lssm_token_logprobs_workspace(r, V, k) for r in range(1, 140)]
    assert sizes == sorted(sizes)
