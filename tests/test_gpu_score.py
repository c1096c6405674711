"""Scoring whole prompts: lssm_engine_score and lssm_cli --score.

Tolerance.  The hidden rows after the last layer come from the engine itself
(set_trace); norm_f and the lm_head are taken in 64 bits from there.  The engine
rounds the normed row and the logits to the activation type, half a step d
each, on top of fp32 sums of d_model terms ((d_model + 8) 2^-24): a logit is off
by at most e = (d + (d_model + 8) 2^-24) sum |h w| / rms + d |logit|, a log
probability by 2 max e + 28 2^-24 (its own logit and the sum's), an entropy by
2 max e (1 + log V) besides its own 84 2^-24 (1 + log V).
"""
import os
import subprocess

import numpy as np
import pytest
import torch

import lite_ssm_amd as L
from lite_ssm_amd.model import DeviceModel, Engine, shape

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CLI = os.path.join(ROOT, "lite_ssm_amd", "lssm_cli")
U = 2.0 ** -24


def expected(m, hidden, tokens):
    """(log p of tokens, entropies, all log p, error bound of a log p) in 64 bits."""
    dt = m.embed.dtype
    h = hidden.double()
    normed = h * m.norm_f.double() / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-5)
    w = m.lm_head.double()
    logits = normed @ w.T
    d = 0.0 if dt is torch.float32 else torch.finfo(dt).eps / 2
    e = (d + (h.shape[-1] + 8) * U) * (normed.abs() @ w.abs().T) + d * logits.abs()
    lp = torch.log_softmax(logits, -1)
    p = torch.exp(lp)
    given = torch.where(tokens < 0, 0.0, lp.gather(1, tokens.clamp(min=0).long()[:, None])[:, 0])
    return given, -(p * lp).sum(-1), lp, 2 * e.max(-1).values + 28 * U


@pytest.mark.parametrize("act,wfmt,B,n,vocab", [
    ("bf16", L.W_Q4_G64, 1, 1, 2048), ("bf16", L.W_Q4_G64, 2, 3, 2048), ("f16", L.W_Q8_G32, 3, 70, 1999),
    ("f16", L.W_DENSE, 2, 9, 2048), ("f32", L.W_DENSE, 2, 40, 1024),
    ("bf16", L.W_Q4_G64, 2, 700, 50280),        # several blocks of rows
    ("bf16", L.W_Q4_G64, 2, 5, 256000),         # rows of several segments
])
def test_engine_scores_a_prompt(ctx, act, wfmt, B, n, vocab):
    code = {"f16": L.F16, "bf16": L.BF16, "f32": L.F32}[act]
    sh = shape("mamba2-130m", n_layer=1, vocab_size=vocab)
    m = DeviceModel(sh, act=code, wfmt=wfmt, seed=3, embed_std=0.1)
    torch.cuda.synchronize()
    eng = Engine(ctx, m, max_batch=B, max_seq=n)
    g = torch.Generator().manual_seed(n)
    ids = torch.randint(0, vocab, (B, n), generator=g, dtype=torch.int32).cuda()
    tokens = torch.cat([ids[:, 1:], torch.full((B, 1), -1, dtype=torch.int32, device="cuda")], 1).contiguous()
    nxt, nxt2 = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2))
    eng.prefill(ids, nxt)
    logits, (conv, ssd) = eng.logits(B), eng.state()
    trace = torch.zeros((sh.n_layer + 1) * B * n, sh.d_model, dtype=m.embed.dtype, device="cuda")
    eng.set_trace(trace)
    eng.reset()
    K = 4
    lp, H = torch.full((B, n), 7.0, device="cuda"), torch.full((B, n), 7.0, device="cuda")
    top, tlp = torch.zeros(B, n, K, dtype=torch.int32, device="cuda"), torch.zeros(B, n, K, device="cuda")
    eng.score(ids, nxt2, tokens, lp, H, top, tlp)
    torch.cuda.synchronize()
    # the prefill that it also is
    assert torch.equal(nxt, nxt2) and torch.equal(eng.logits(B), logits)
    assert torch.equal(eng.state()[0], conv) and torch.equal(eng.state()[1], ssd)
    hidden = trace[sh.n_layer * B * n:]
    given, entropy, all_lp, err = expected(m, hidden, tokens.reshape(-1))
    assert bool(((lp.reshape(-1).double() - given).abs() <= err).all())
    V = float(np.log(vocab))
    assert bool(((H.reshape(-1).double() - entropy).abs() <= (err + 84 * U) * (1 + V)).all())
    # alternatives: in order, and each as likely as the true one of its place
    t = tlp.reshape(-1, K).double()
    assert bool((t[:, 1:] <= t[:, :-1]).all())
    best = all_lp.topk(K, -1).values
    assert bool(((t - best).abs() <= err[:, None]).all())
    assert bool(((t - all_lp.gather(1, top.reshape(-1, K).long())).abs() <= err[:, None]).all())
    # the last position's alternatives are the prefill's logits: greedy id first
    assert torch.equal(top[:, -1, 0], nxt)
    eng.set_trace(None)
    # outputs left out, and a second call
    eng.score(ids, nxt2, entropy=H)
    eng.close()


@pytest.mark.parametrize("B,n", [(2, 4096), (1, 8192)])
def test_a_prefill_of_two_halves_is_scored(ctx, B, n):
    """8192 rows run as two halves on two streams (batch, or time), with a trace
    buffer set as one.  The two forms' logits are each within 2e-2 of the largest
    of the reference's, so their log probabilities within 8e-2 of it; a row
    that is not its position's is off by several units."""
    sh = shape("mamba2-130m", n_layer=2, vocab_size=1024)
    m = DeviceModel(sh, act=L.BF16, wfmt=L.W_Q4_G64, seed=3, embed_std=0.1)
    torch.cuda.synchronize()
    eng = Engine(ctx, m, max_batch=B, max_seq=n)
    g = torch.Generator().manual_seed(n)
    ids = torch.randint(0, 1024, (B, n), generator=g, dtype=torch.int32).cuda()
    nxt = torch.zeros(B, dtype=torch.int32, device="cuda")
    lp, H = ([torch.full((B, n), 7.0, device="cuda") for _ in range(2)] for _ in range(2))
    top, tlp = torch.zeros(B, n, 1, dtype=torch.int32, device="cuda"), torch.zeros(B, n, 1, device="cuda")
    eng.score(ids, nxt, ids, lp[0], H[0], top, tlp)
    torch.cuda.synchronize()
    assert torch.equal(top[:, -1, 0], nxt)
    trace = torch.zeros((sh.n_layer + 1) * B * n, sh.d_model, dtype=torch.bfloat16, device="cuda")
    eng.set_trace(trace)
    eng.reset()
    eng.score(ids, nxt, ids, lp[1], H[1])
    torch.cuda.synchronize()
    given, entropy, all_lp, err = expected(m, trace[sh.n_layer * B * n:], ids.reshape(-1))
    assert bool(((lp[1].reshape(-1).double() - given).abs() <= err).all())
    largest = float((all_lp - all_lp.mean(-1, keepdim=True)).abs().max())
    assert float((lp[0] - lp[1]).abs().max()) <= 8e-2 * largest < 2.0
    eng.set_trace(None)
    eng.close()


def test_engine_score_refuses(ctx):
    sh = shape("mamba2-130m", n_layer=1, vocab_size=128)
    m = DeviceModel(sh, act=L.BF16, wfmt=L.W_Q4_G64, seed=3)
    torch.cuda.synchronize()
    eng = Engine(ctx, m, max_batch=1, max_seq=8)
    ids = torch.zeros(1, 8, dtype=torch.int32, device="cuda")
    nxt = torch.zeros(1, dtype=torch.int32, device="cuda")
    f = torch.zeros(8 * 200, device="cuda")
    p = f.data_ptr()

    def bad(text, ids=ids.data_ptr(), B=1, n=8, nx=nxt.data_ptr(), t=p, lp=p, H=p, ti=None, tl=None, k=0):
        assert L.lib.lssm_engine_score(eng.h, ids, B, n, nx, t, lp, H, ti, tl, k) == 1
        assert text in L.lib.lssm_last_error().decode()
    bad("L must be", n=9)
    bad("L must be", n=0)
    bad("batch out of range", B=2)
    bad("null ids", ids=None)
    bad("null ids", nx=None)
    bad("go together", t=None)
    bad("go together", lp=None)
    bad("top_k must be", k=65, ti=p, tl=p)
    bad("top_k must be", k=129, ti=p, tl=p)
    bad("top_k without", k=3)
    bad("4-byte aligned", H=p + 2)
    assert L.lib.lssm_engine_score(None, None, 1, 1, None, None, None, None, None, None, 0) == 1
    # a token past the vocabulary is reported, the others are scored
    t = torch.tensor([1, 128, 2, 3, 4, 5, 6, -1], dtype=torch.int32, device="cuda")
    with pytest.raises(L.LssmError, match="not below the vocabulary"):
        eng.score(ids, nxt, t, f[:8])
    assert torch.isnan(f[:8]).tolist() == [False, True] + [False] * 6
    eng.close()


def test_cli_scores_a_prompt(ctx, tmp_path):
    from lite_ssm_amd import ssm as S
    path = tmp_path / "m.ssm"
    S.write_random(path, shape("mamba2-130m", n_layer=2, vocab_size=2048), L.BF16, L.W_Q4_G64, seed=4)
    prompt = [5, 77, 1023, 9, 2047, 0, 314, 15, 92, 600, 11]
    r = subprocess.run([CLI, "--model", str(path), "--score", "--top-logprobs", "3", "--input-ids", ",".join(map(str, prompt))],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    lines = [ln.split() for ln in r.stdout.splitlines()]
    assert [int(ln[0]) for ln in lines] == prompt[1:]
    n = len(prompt)
    with S.SSMFile(path) as f:
        fm = f.model(ctx)
        eng = Engine(ctx, fm, 1, max(n, fm.shape.chunk_size))
        ids = torch.tensor([prompt], dtype=torch.int32).cuda()
        tokens = torch.tensor([prompt[1:] + [-1]], dtype=torch.int32).cuda()
        nxt = torch.zeros(1, dtype=torch.int32, device="cuda")
        lp, H = torch.zeros(1, n, device="cuda"), torch.zeros(1, n, device="cuda")
        top, tlp = torch.zeros(1, n, 3, dtype=torch.int32, device="cuda"), torch.zeros(1, n, 3, device="cuda")
        eng.score(ids, nxt, tokens, lp, H, top, tlp)
        torch.cuda.synchronize()
        eng.close()
    for i, ln in enumerate(lines):
        assert abs(float(ln[1]) - float(lp[0, i])) < 1e-6            # printed with six digits
        alt = [a.split(":") for a in ln[2:]]
        assert [int(a) for a, _ in alt] == top[0, i].tolist()
        assert all(abs(float(v) - float(tlp[0, i, k])) < 1e-6 for k, (_, v) in enumerate(alt))
    total = float(lp[0, :n - 1].double().sum())
    assert f"log probability {total:.3f}" in r.stderr or abs(float(r.stderr.split("log probability ")[1].split()[0]) - total) < 1e-3
