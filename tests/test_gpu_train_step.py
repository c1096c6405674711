"""The scan, its gradient and the loss together, as a training step uses them: a
small recurrent language model whose products with weights are torch's and
whose scan, log probabilities and gradients are the library's, in fp32, against
torch's differentiation of the same model in 64 bits.

Tolerance.  Five stages of fp32 arithmetic (projections, scan, logits and loss,
scan's gradient, weight gradients), each off by at most 400 2^-24 of its terms'
size (see test_gpu_ssd_bwd.py), added up: 1.2e-4 of the gradient's size, with a
factor of four for terms that cancel in it.
"""
import pytest
import torch

import lite_ssm_amd as L
from ssd_bwd_ref import forward

pytestmark = pytest.mark.gpu


def model(seed, V, d, H, P, G, N):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return dict(embed=r(V, d), wx=r(d, H * P) / d ** 0.5, wb=r(d, G * N) / (d * N) ** 0.5, wc=r(d, G * N) / (d * N) ** 0.5,
                wd=r(d, H) / d ** 0.5, dt_bias=r(H) - 2, A_log=torch.log(1 + 15 * torch.rand(H, generator=g)), D=r(H),
                head=r(V, H * P) / (H * P) ** 0.5)


def parts(w, ids, H, P, G, N):
    b, n = ids.shape
    x = w["embed"][ids]
    return dict(X=(x @ w["wx"]).reshape(b, n, H, P), B=(x @ w["wb"]).reshape(b, n, G, N),
                C=(x @ w["wc"]).reshape(b, n, G, N), dt=x @ w["wd"])


@pytest.mark.parametrize("b,n,H,P,G,N,V", [(2, 50, 4, 64, 2, 128, 500), (1, 130, 3, 32, 1, 64, 301)])
def test_gradients_of_a_step(ctx, b, n, H, P, G, N, V):
    d = 48
    w = model(n, V, d, H, P, G, N)
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, V, (b, n), generator=g)
    targets = torch.randint(0, V, (b, n), generator=g)
    targets[:, :5] = -1                                   # a prompt without loss
    count = int((targets >= 0).sum())
    # in 64 bits, by torch
    leaves = {k: v.double().requires_grad_() for k, v in w.items()}
    v = dict(parts(leaves, ids, H, P, G, N), dt_bias=leaves["dt_bias"], A_log=leaves["A_log"], D=leaves["D"],
             state=torch.zeros(b, H, P, N, dtype=torch.float64))
    y, _ = forward(v, 1e-6, 1e6)
    lp = torch.log_softmax(y.reshape(b * n, H * P) @ leaves["head"].T, -1)
    t = targets.reshape(-1)
    loss = -lp[torch.arange(b * n), t.clamp(min=0)][t >= 0].mean()
    loss.backward()

    # fp32, by the library
    c = {k: x.cuda() for k, x in w.items()}
    p = {k: x.contiguous() for k, x in parts(c, ids.cuda(), H, P, G, N).items()}
    kw = dict(device="cuda")
    state, Y = torch.zeros(b, H, P, N, **kw), torch.empty(b, n, H, P, **kw)
    dims = L.SSDDims(n, H, P, N, G, min(64, n), 1e-6, 1e6, 1)
    torch.cuda.synchronize()
    ctx.ssd_chunked(p["X"], p["B"], p["C"], p["dt"], c["dt_bias"], c["A_log"], c["D"], Y, state, b, dims, L.F32)
    rows = Y.reshape(b * n, H * P)
    logits = rows @ c["head"].T
    tok = t.to(torch.int32).cuda()
    gl = torch.where(tok >= 0, -1.0 / count, 0.0).float()
    out, ent, st = torch.empty(b * n, **kw), torch.empty(b * n, **kw), torch.empty(b * n, 2, **kw)
    torch.cuda.synchronize()
    ctx.token_logprobs_grad(logits, tok, gl, None, out, ent, st, logits, b * n, V, L.F32)       # in place
    got_loss = -float(out.sum()) / count
    d_head, dY = logits.T @ rows, (logits @ c["head"]).reshape(b, n, H, P).contiguous()
    o = {k: torch.empty_like(p[k]) for k in p}
    o.update({k: torch.empty(H, **kw) for k in ("dt_bias", "A_log", "D")})
    ws = torch.empty(ctx.ssd_chunked_bwd_workspace(b, dims, L.F32), dtype=torch.uint8, **kw)
    torch.cuda.synchronize()
    ctx.ssd_chunked_bwd(p["X"], p["B"], p["C"], p["dt"], c["dt_bias"], c["A_log"], c["D"], None, dY, None, o["X"], o["B"],
                        o["C"], o["dt"], o["dt_bias"], o["A_log"], o["D"], None, b, dims, L.F32, ws)
    x = c["embed"][ids.cuda()].reshape(b * n, d)
    flat = {k: o[k].reshape(b * n, -1) for k in p}
    dx = sum(flat[k] @ c[m].T for k, m in (("X", "wx"), ("B", "wb"), ("C", "wc"), ("dt", "wd")))
    d_embed = torch.zeros_like(c["embed"]).index_add_(0, ids.cuda().reshape(-1), dx)
    got = dict(embed=d_embed, wx=x.T @ flat["X"], wb=x.T @ flat["B"], wc=x.T @ flat["C"], wd=x.T @ flat["dt"],
               dt_bias=o["dt_bias"], A_log=o["A_log"], D=o["D"], head=d_head)
    assert abs(got_loss - float(loss.detach())) < 1.2e-4 * abs(float(loss.detach()))
    for k, leaf in leaves.items():
        err = float((got[k].double().cpu() - leaf.grad).norm())
        assert err < 4 * 1.2e-4 * float(leaf.grad.norm()), (k, err / float(leaf.grad.norm()))
