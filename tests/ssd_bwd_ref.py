"""The scan's gradients in 64 bits, by its recurrences token by token (CPU), and
the sums of absolute terms that rounding errors are measured against."""
import torch

NAMES = ("dX", "dB", "dC", "d_dt", "d_dt_bias", "dA_log", "dD", "d_state0")


def forward(v, dt_min, dt_max):
    """Y and the final state; v: X, B, C, dt, dt_bias, A_log, D, state (64 bits)."""
    b, L, H, P = v["X"].shape
    hpg = H // v["B"].shape[2]
    soft = torch.logaddexp(v["dt"] + v["dt_bias"], torch.zeros((), dtype=torch.float64))
    dt, A = soft.clamp(dt_min, dt_max), -torch.exp(v["A_log"])
    h, ys = v["state"], []
    for t in range(L):
        B, C = (v[k][:, t].repeat_interleave(hpg, 1)[:, :, None, :] for k in ("B", "C"))
        h = torch.exp(A * dt[:, t])[..., None, None] * h + (dt[:, t][..., None] * v["X"][:, t])[..., None] * B
        ys.append((h * C).sum(-1) + v["D"][:, None] * v["X"][:, t])
    return (torch.stack(ys, 1) if ys else v["X"] * 0), h


def grads(v, dt_min, dt_max, absolute=False):
    """All gradients for dY, d_state in v.  absolute: of |inputs|, every term of
    every sum added with a positive sign."""
    v = {k: t.double().cpu() for k, t in v.items()}
    raw = v["dt"] + v["dt_bias"]
    soft = torch.logaddexp(raw, torch.zeros((), dtype=torch.float64))
    dt, A = soft.clamp(dt_min, dt_max), -torch.exp(v["A_log"])
    slope = torch.sigmoid(raw) * ((soft >= dt_min) & (soft <= dt_max))
    if absolute:
        v = {k: t if k in ("dt", "dt_bias", "A_log") else t.abs() for k, t in v.items()}
    mag = A.abs() if absolute else A
    x, dy = v["X"], v["dY"]
    b, L, H, P = x.shape
    G, N = v["B"].shape[2:]
    hpg = H // G
    decay = torch.exp(A * dt)
    heads = lambda k, t: v[k][:, t].repeat_interleave(hpg, 1)[:, :, None, :]  # noqa: E731
    hs = [v["state"]]
    for t in range(L):
        hs.append(decay[:, t][..., None, None] * hs[-1] + (dt[:, t][..., None] * x[:, t])[..., None] * heads("B", t))
    o = dict(dX=torch.zeros_like(x), dB=torch.zeros_like(v["B"]), dC=torch.zeros_like(v["C"]), d_dt=torch.zeros_like(dt))
    dA = torch.zeros(H, dtype=torch.float64)
    g = v["d_state"]
    for t in reversed(range(L)):
        g = g + dy[:, t][..., None] * heads("C", t)
        o["dC"][:, t] = (hs[t + 1] * dy[:, t][..., None]).sum(2).reshape(b, G, hpg, N).sum(2)
        o["dB"][:, t] = (dt[:, t][..., None] * (g * x[:, t][..., None]).sum(2)).reshape(b, G, hpg, N).sum(2)
        gb = (g * heads("B", t)).sum(-1)
        o["dX"][:, t] = dt[:, t][..., None] * gb + v["D"][:, None] * dy[:, t]
        g = decay[:, t][..., None, None] * g
        a = (g * hs[t]).sum((-1, -2))
        o["d_dt"][:, t] = ((gb * x[:, t]).sum(-1) + mag * a) * slope[:, t]
        dA += (dt[:, t] * a).sum(0)
    return dict(o, d_dt_bias=o["d_dt"].sum((0, 1)), dA_log=mag * dA, dD=(x * dy).sum((0, 1, 3)), d_state0=g)
