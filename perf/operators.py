"""Scoring and training operators: log probabilities of tokens with their
gradient, and the gradient of the SSD scan, as cases to time and check.

A case is a dict of plain values with a "kind":

  logprobs   log probabilities of given tokens, entropies and the top_k best
             alternatives of rows of logits (scoring a prompt, or the tokens a
             decode step chose)
  nll        the same values together with the gradient to the logits, where the
             upstream gradients are known beforehand (mean NLL training)
  policy     log probabilities first, the upstream gradient computed from them
             (a policy ratio), then the gradient to the logits
  ssd_bwd    all gradients of the Mamba-2 scan of one layer

Where `own` is false, run() computes the plain form with torch in 32 bits (the
step sizes and decays in 64); where it is true, it calls the library.
"""
import functools
import math

import torch

own = False

DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# heads, head size, groups, state size of one layer; vocabulary
MODELS = {"mamba2-130m": (24, 64, 1, 128), "mamba2-2.7b": (80, 64, 1, 128), "mamba2-8b": (128, 64, 8, 128)}
DT_MIN, DT_MAX, CHUNK = 1e-6, 1e6, 64
# limits of a drawn case: those of the largest listed ones
MAX_LOGIT_BYTES, MAX_SCAN, MAX_SCAN_F32 = 8e8, 4 * 4096 * 80 * 64 * 128, 2048 * 24 * 64 * 128


def listed():
    return [
        # one sequence's chosen token after a decode step of the smallest model,
        # with five alternatives: the smallest call, where latency counts
        dict(name="logprobs_decode_1", kind="logprobs", rows=1, vocab=50280, act="f16", top_k=5),
        # a serving batch at the widest vocabulary, twenty alternatives
        dict(name="logprobs_decode_32", kind="logprobs", rows=32, vocab=256000, act="bf16", top_k=20),
        # a ragged prompt scored by an fp32 model, a padded (odd) vocabulary
        dict(name="logprobs_fp32_301", kind="logprobs", rows=301, vocab=50281, act="f32", top_k=8),
        # a batch of long documents scored for their likelihood: the largest
        dict(name="logprobs_score_8000", kind="logprobs", rows=7999, vocab=50280, act="bf16", top_k=0),
        # a training batch's loss and gradient
        dict(name="nll_2048", kind="nll", rows=2048, vocab=50280, act="bf16"),
        # the same at the widest vocabulary: a row does not fit on a CU
        dict(name="nll_wide_700", kind="nll", rows=700, vocab=256000, act="bf16"),
        # a policy gradient with an entropy bonus over short answers
        dict(name="policy_517", kind="policy", rows=517, vocab=50280, act="f16"),
        # the fp32 scan of the 130M layer at 512 tokens, as it is checked against its source
        dict(name="ssd_bwd_fp32_512", kind="ssd_bwd", model="mamba2-130m", batch=1, tokens=512, act="f32", state=True),
        # one short ragged sentence of the smallest model
        dict(name="ssd_bwd_short_37", kind="ssd_bwd", model="mamba2-130m", batch=1, tokens=37, act="f16", state=False),
        # two ragged documents through an 8B layer (eight groups)
        dict(name="ssd_bwd_8b_2x1777", kind="ssd_bwd", model="mamba2-8b", batch=2, tokens=1777, act="bf16", state=True),
        # one long sequence through a 2.7B layer
        dict(name="ssd_bwd_4096", kind="ssd_bwd", model="mamba2-2.7b", batch=1, tokens=4096, act="bf16", state=False),
        # a training batch of long sequences through the same layer: the largest
        dict(name="ssd_bwd_4x4096", kind="ssd_bwd", model="mamba2-2.7b", batch=4, tokens=4096, act="bf16", state=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    """One case of the same ranges, sizes over their logarithm."""
    kind = rng.choice(("logprobs", "logprobs", "nll", "policy", "ssd_bwd", "ssd_bwd", "ssd_bwd"))
    act = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind != "ssd_bwd":
        vocab = rng.choice((50280, 256000, _log_int(rng, 500, 256000)))
        most = MAX_LOGIT_BYTES / (vocab * (4 if act == "f32" else 2) * (1 if kind == "logprobs" else 2))
        case = dict(kind=kind, rows=_log_int(rng, 1, min(8192, int(most))), vocab=vocab, act=act)
        return dict(case, top_k=rng.choice((0, 1, 5, 20))) if kind == "logprobs" else case
    model = rng.choice(tuple(MODELS) + ("other",))
    case = dict(kind=kind, model=model, act=act, state=rng.random() < 0.5, batch=_log_int(rng, 1, 8))
    if model == "other":
        G = rng.choice((1, 2, 4))
        case.update(heads=G * rng.randint(1, 8), head=rng.choice((32, 64, 80, 128)), groups=G,
                    dstate=rng.choice((16, 64, 128, 200)))
    H, P, G, N = _dims(case)
    most = (MAX_SCAN_F32 if act == "f32" else MAX_SCAN) / (H * P * N * case["batch"])
    return dict(case, tokens=_log_int(rng, 1, min(16384, max(1, int(most)))))


def _dims(case):
    if case["model"] == "other":
        return case["heads"], case["head"], case["groups"], case["dstate"]
    return MODELS[case["model"]]


# --------------------------------------------------------------------------- inputs
def _logit_inputs(case, seed):
    """Logits of a trained model's spread: the given tokens are likely ones more
    often than not.  The last entries of a padded vocabulary are masked (-inf),
    and some positions (a prompt's) have no token to score (-1)."""
    g = torch.Generator(device="cuda").manual_seed(1 + seed)
    M, V = case["rows"], case["vocab"]
    x = torch.randn(M, V, generator=g, device="cuda", dtype=torch.float32 if case["act"] == "f32" else torch.float16)
    x = x.mul_(2.5).to(DTYPE[case["act"]])
    tokens = torch.randint(0, V - 8, (M,), generator=g, device="cuda")
    boost = torch.rand(M, generator=g, device="cuda") * 16 - 4
    at = torch.arange(M, device="cuda")
    x[at, tokens] = (x[at, tokens].float() + boost).to(x.dtype)
    x[:, V - 8:] = -math.inf
    none = torch.rand(M, generator=g, device="cuda") < 0.15
    none[0] = False
    st = dict(logits=x, tokens=torch.where(none, -1, tokens).to(torch.int32))
    if case["kind"] == "nll":
        n = (~none).sum().clamp(min=1)
        st["g_logprob"] = torch.where(none, 0.0, -1.0 / n).float()
    if case["kind"] == "policy":
        st["old"] = -torch.rand(M, generator=g, device="cuda") * 10
        st["advantage"] = torch.randn(M, generator=g, device="cuda")
        st["g_entropy"] = torch.full((M,), -0.01, device="cuda")
    return st


def _ssd_inputs(case, seed):
    """X, B, C as the conv's SiLU leaves them in scale; dt, A and D as Mamba-2
    sets them up; the gradients of the outputs of unit size."""
    g, dt = torch.Generator(device="cuda").manual_seed(1 + seed), DTYPE[case["act"]]
    H, P, G, N = _dims(case)
    b, n = case["batch"], case["tokens"]

    def randn(*size):
        return torch.randn(*size, generator=g, device="cuda")

    step = torch.exp(torch.rand(H, generator=g, device="cuda") * math.log(100.0) + math.log(1e-3))
    st = dict(X=randn(b, n, H, P).to(dt), B=(randn(b, n, G, N) / N ** 0.5).to(dt), C=(randn(b, n, G, N) / N ** 0.5).to(dt),
              dt=(0.5 * randn(b, n, H)).to(dt), dt_bias=(step + torch.log(-torch.expm1(-step))).to(dt),
              A_log=torch.log(1 + 15 * torch.rand(H, generator=g, device="cuda")).to(dt),
              D=(1 + 0.1 * randn(H)).to(dt), dY=randn(b, n, H, P).to(dt))
    # the state entering the scan and the gradient of the one that leaves it
    st["state"] = randn(b, H, P, N) if case["state"] else None
    st["d_state"] = 0.1 * randn(b, H, P, N) if case["state"] else None
    return st


def prepare(case, seed):
    """The inputs, and the output buffers that such a program keeps."""
    kw = dict(device="cuda")
    if case["kind"] == "ssd_bwd":
        st = _ssd_inputs(case, seed)
        for k in ("X", "B", "C", "dt", "dt_bias", "A_log", "D"):
            st["d_" + k] = torch.empty_like(st[k])
        H, P, G, N = _dims(case)
        st["d_state0"] = torch.empty(case["batch"], H, P, N, **kw)
    else:
        st = _logit_inputs(case, seed)
        M, k = case["rows"], case.get("top_k", 0)
        st.update(logprob=torch.empty(M, **kw), entropy=torch.empty(M, **kw), stats=torch.empty(M, 2, **kw),
                  top_ids=torch.empty(M, k, dtype=torch.int32, **kw), top_logprobs=torch.empty(M, k, **kw))
        if case["kind"] != "logprobs":
            st["d_logits"] = torch.empty_like(st["logits"])
    return dict(st, case=dict(case))


# --------------------------------------------------------------------------- one pass
def run(st):
    if own:
        return _own(st)
    kind = st["case"]["kind"]
    return _plain_ssd(st) if kind == "ssd_bwd" else _plain_logits(st, kind)


@functools.lru_cache(None)
def _ctx():
    """The program's one context; its batch stays open, as calls only enqueue within one."""
    import lite_ssm_amd as L
    stream = torch.cuda.Stream()
    ctx = L.Ctx(stream=stream.cuda_stream)
    ctx.begin_batch()
    return L, ctx, stream


def _own(st):
    L, ctx, stream = _ctx()
    case = st["case"]
    act = {"f16": L.F16, "bf16": L.BF16, "f32": L.F32}[case["act"]]
    if case["kind"] == "ssd_bwd":
        H, P, G, N = _dims(case)
        dims = L.SSDDims(case["tokens"], H, P, N, G, CHUNK, DT_MIN, DT_MAX, 1)
        if "ws" not in st:
            st["ws"] = torch.empty(ctx.ssd_chunked_bwd_workspace(case["batch"], dims, act), dtype=torch.uint8, device="cuda")
        ctx.ssd_chunked_bwd(st["X"], st["B"], st["C"], st["dt"], st["dt_bias"], st["A_log"], st["D"], st["state"],
                            st["dY"], st["d_state"], st["d_X"], st["d_B"], st["d_C"], st["d_dt"], st["d_dt_bias"],
                            st["d_A_log"], st["d_D"], st["d_state0"], case["batch"], dims, act, st["ws"])
        return {k: st[k] for k in ("d_X", "d_B", "d_C", "d_dt", "d_dt_bias", "d_A_log", "d_D", "d_state0")}
    M, V, k = case["rows"], case["vocab"], case.get("top_k", 0)
    if "ws" not in st:
        st["ws"] = torch.empty(ctx.token_logprobs_workspace(M, V, k), dtype=torch.uint8, device="cuda")
    out = {n: st[n] for n in ("logprob", "entropy")}
    if case["kind"] == "nll":
        ctx.token_logprobs_grad(st["logits"], st["tokens"], st["g_logprob"], None, st["logprob"], st["entropy"],
                                st["stats"], st["d_logits"], M, V, act, st["ws"])
        return dict(out, d_logits=st["d_logits"])
    ctx.token_logprobs(st["logits"], st["tokens"], st["logprob"], st["entropy"], st["stats"], st["top_ids"],
                       st["top_logprobs"], M, V, k, act, st["ws"])
    if case["kind"] == "logprobs":
        return dict(out, top_ids=st["top_ids"], top_logprobs=st["top_logprobs"])
    with torch.cuda.stream(stream):
        g = _policy(st, st["logprob"])
        ctx.token_logprobs_bwd(st["logits"], st["tokens"], st["stats"], st["entropy"], g, st["g_entropy"],
                               st["d_logits"], M, V, act)
    return dict(out, d_logits=st["d_logits"])


def _policy(st, logprob):
    """Gradient of -(ratio * advantage) to the log probability."""
    ratio = torch.exp(torch.clamp(logprob - st["old"], max=3.0))
    return torch.where(st["tokens"] >= 0, -ratio * st["advantage"], 0.0)


# --------------------------------------------------------------------------- plain form
def _plain_logits(st, kind):
    x, tokens = st["logits"].float(), st["tokens"].long()
    m = x.max(-1, keepdim=True).values
    d = x - m
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    ls = torch.log(total)
    p = e / total
    entropy = ls[:, 0] - torch.where(p > 0, p * d, 0.0).sum(-1)
    given = tokens >= 0
    at = tokens.clamp(min=0)[:, None]
    logprob = torch.where(given, (d - ls).gather(1, at)[:, 0], 0.0)
    out = dict(logprob=logprob, entropy=entropy)
    if kind == "logprobs":
        k = st["top_ids"].shape[1]
        if k == 0:
            return dict(out, top_ids=st["top_ids"], top_logprobs=st["top_logprobs"])
        # equal values: the lowest index first (value and place in one whole number)
        bits = st["logits"].float().view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
        key = order * 2 ** 31 + (2 ** 31 - 1 - torch.arange(x.shape[1], device=x.device))
        ids = 2 ** 31 - 1 - (torch.topk(key, k, dim=-1).values & (2 ** 31 - 1))
        return dict(out, top_ids=ids.to(torch.int32), top_logprobs=(d - ls).gather(1, ids))
    g = st["g_logprob"] if kind == "nll" else _policy(st, logprob)
    grad = -g[:, None] * p
    if kind == "policy":
        grad = grad - st["g_entropy"][:, None] * torch.where(p > 0, p * (d - ls + entropy[:, None]), 0.0)
    grad.scatter_add_(1, at, torch.where(given, g, 0.0)[:, None])
    return dict(out, d_logits=grad.to(st["logits"].dtype))


def _plain_ssd(st):
    """The chunked form: 64 tokens at a time as products of matrices, the states
    between chunks as one product with the chunks' decays."""
    case, act = st["case"], st["X"].dtype
    H, P, G, N = _dims(case)
    b, n, Q = case["batch"], case["tokens"], CHUNK
    nc = -(-n // Q)
    raw = st["dt"].double() + st["dt_bias"].double()
    soft = torch.log1p(torch.exp(-raw.abs())) + raw.clamp(min=0)
    dt = soft.clamp(DT_MIN, DT_MAX)
    slope = torch.where((soft >= DT_MIN) & (soft <= DT_MAX), torch.sigmoid(raw), 0.0)
    A = -torch.exp(st["A_log"].double())

    def chunks(v):  # [b, n, h, ...] -> [b, h, nc, Q, ...], zeros behind the end
        pad = torch.zeros(b, nc * Q - n, *v.shape[2:], dtype=v.dtype, device=v.device)
        v = torch.cat([v, pad], 1).reshape(b, nc, Q, *v.shape[2:])
        return v.movedim(3, 1).contiguous()

    def rows(v):    # back to [b, n, h, ...]
        return v.movedim(1, 3).reshape(b, nc * Q, v.shape[1], *v.shape[4:])[:, :n]

    def heads(v):   # a group's rows for each of its heads
        return v.repeat_interleave(H // G, 1)

    def group_sum(v):
        return v.reshape(b, G, H // G, *v.shape[2:]).sum(2)

    mt = lambda v: v.transpose(-1, -2).contiguous()  # noqa: E731
    x, dy = chunks(st["X"].float()), chunks(st["dY"].float())
    B, C = heads(chunks(st["B"].float())), heads(chunks(st["C"].float()))
    dtc = chunks(dt)
    cum = (dtc * A[:, None, None]).cumsum(-1)                                   # [b, H, nc, Q], 64 bits
    tot = cum[..., -1]
    dtf = dtc.float()
    decay = torch.exp((cum[..., :, None] - cum[..., None, :]).clamp(max=0.0)).float().tril()
    into, outof = torch.exp(cum).float(), torch.exp(tot[..., None] - cum).float()

    # states: each chunk's own part, then all chunks' parts decayed to each border
    h_own = torch.matmul(mt(x * (outof * dtf)[..., None]), B)                   # [b, H, nc, P, N]
    g_own = torch.matmul(mt(dy * into[..., None]), C)
    zero = torch.zeros(b, H, 1, P, N, device=x.device)
    h_all = torch.cat([zero if st["state"] is None else st["state"][:, :, None], h_own], 2)
    g_all = torch.cat([g_own, zero if st["d_state"] is None else st["d_state"][:, :, None]], 2)
    border = torch.cat([torch.zeros_like(tot[..., :1]), tot.cumsum(-1)], -1)    # decay from the start to border c
    across = torch.exp((border[..., :, None] - border[..., None, :]).clamp(max=0.0)).float().tril()
    h_at = torch.matmul(across, h_all.reshape(b, H, nc + 1, P * N)).reshape(b, H, nc + 1, P, N)
    g_at = torch.matmul(mt(across), g_all.reshape(b, H, nc + 1, P * N)).reshape(b, H, nc + 1, P, N)
    h0, g1 = h_at[:, :, :nc], g_at[:, :, 1:]

    S = torch.matmul(dy, mt(x)) * decay                                         # [t, j], without dt_j
    CB = torch.matmul(C, mt(B)) * decay
    dC = into[..., None] * torch.matmul(dy, h0) + torch.matmul(S * dtf[..., None, :], B)
    dB = outof[..., None] * torch.matmul(x, g1) + torch.matmul(mt(S), C)        # without dt
    dx = outof[..., None] * torch.matmul(B, mt(g1)) + torch.matmul(mt(CB), dy)  # without dt
    direct = (x * dx).sum(-1)
    v, u = (C * dC).sum(-1), direct * dtf
    edge = (g1 * h_at[:, :, 1:]).sum((-1, -2))
    da = (edge[..., None] + (v - u).flip(-1).cumsum(-1).flip(-1))
    ddt = direct + A.float()[:, None, None] * da
    d_dt = rows(ddt) * slope.float()
    return dict(
        d_X=(rows(dx * dtf[..., None]) + st["D"].float()[:, None] * st["dY"].float()).to(act),
        d_B=rows(group_sum(dB * dtf[..., None])).to(act), d_C=rows(group_sum(dC)).to(act),
        d_dt=d_dt.to(act), d_dt_bias=d_dt.double().sum((0, 1)).to(act),
        d_A_log=(A * (da * dtf).double().sum((0, 2, 3))).to(act),
        d_D=(st["dY"].float() * st["X"].float()).sum(-1).double().sum((0, 1)).to(act),
        d_state0=g_at[:, :, 0].contiguous())


# --------------------------------------------------------------------------- work
def work(case):
    es = 4 if case["act"] == "f32" else 2
    if case["kind"] == "ssd_bwd":
        H, P, G, N = _dims(case)
        T, state = case["batch"] * case["tokens"], case["batch"] * H * P * N
        # X, dY in, dX out; B, C in, dB, dC out; dt in and out; a state in, one out
        rows = es * T * (3 * H * P + 4 * G * N + 2 * H)
        # the recurrences of h and G, and their products dC, dB, dx, each 2 N P a head and token
        return dict(bytes=rows + 4.0 * state * (3 if case["state"] else 1), flops=10.0 * T * H * P * N)
    M, V, k = case["rows"], case["vocab"], case.get("top_k", 0)
    grad = case["kind"] != "logprobs"
    return dict(bytes=float(es * M * V * (2 if grad else 1) + M * (12 + 8 * k)), flops=(8.0 if grad else 4.0) * M * V)


# --------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    if case["kind"] == "ssd_bwd":
        return _exact_ssd(case, _ssd_inputs(case, seed))
    st = _logit_inputs(case, seed)
    parts = [_exact_rows(case, {k: v[r:r + 256] for k, v in st.items()}) for r in range(0, case["rows"], 256)]
    return {k: None if parts[0][k] is None else torch.cat([p[k] for p in parts]) for k in parts[0]}


def _exact_rows(case, st):
    x, tokens = st["logits"].double(), st["tokens"].long()
    lp = x - torch.logsumexp(x, -1, keepdim=True)
    p = torch.exp(lp)
    entropy = -torch.nan_to_num(p * lp, nan=0.0).sum(-1)
    given = tokens >= 0
    logprob = torch.where(given, lp.gather(1, tokens.clamp(min=0)[:, None])[:, 0], 0.0)
    if case["kind"] == "logprobs":
        best = torch.sort(lp, dim=-1, descending=True).values if case["top_k"] else lp
        return dict(logprob=logprob, entropy=entropy, top_ids=None, top_logprobs=best[:, :case["top_k"]])
    if case["kind"] == "nll":
        g, ge = st["g_logprob"].double(), torch.zeros_like(entropy)
    else:
        ratio = torch.exp(torch.clamp(logprob - st["old"].double(), max=3.0))
        g, ge = torch.where(given, -ratio * st["advantage"].double(), 0.0), st["g_entropy"].double()
    onehot = torch.zeros_like(x)
    onehot[torch.arange(len(x), device=x.device)[given], tokens[given]] = 1.0
    grad = g[:, None] * (onehot - p) - ge[:, None] * torch.nan_to_num(p * (lp + entropy[:, None]), nan=0.0)
    return dict(logprob=logprob, entropy=entropy, d_logits=grad)


def _exact_ssd(case, st):
    """The recurrences token by token: forward with the state kept every 64
    tokens, then backwards, each span's states recomputed."""
    H, P, G, N = _dims(case)
    b, n, span = case["batch"], case["tokens"], 64
    x, dy = st["X"].double(), st["dY"].double()
    Bm, Cm = st["B"].double(), st["C"].double()
    raw = st["dt"].double() + st["dt_bias"].double()
    soft = torch.nn.functional.softplus(raw, threshold=1e9)
    dt = soft.clamp(DT_MIN, DT_MAX)
    A = -torch.exp(st["A_log"].double())
    kw = dict(dtype=torch.float64, device="cuda")
    h = torch.zeros(b, H, P, N, **kw) if st["state"] is None else st["state"].double()
    G1 = torch.zeros(b, H, P, N, **kw) if st["d_state"] is None else st["d_state"].double()
    hpg = H // G

    def step(h, t):
        decay = torch.exp(A * dt[:, t])[..., None, None]
        row = Bm[:, t].repeat_interleave(hpg, 1)[:, :, None, :]
        return decay * h + (dt[:, t][..., None] * x[:, t])[..., None] * row

    kept = []
    for t in range(n):
        if t % span == 0:
            kept.append(h)
        h = step(h, t)
    d_X, d_B, d_C, d_dt = torch.empty_like(x), torch.empty_like(Bm), torch.empty_like(Cm), torch.empty_like(dt)
    d_A = torch.zeros(H, **kw)
    for c in reversed(range(len(kept))):
        lo, hi = c * span, min(n, (c + 1) * span)
        before, h = [], kept.pop()
        for t in range(lo, hi):
            before.append(h)
            h = step(h, t)
        for t in reversed(range(lo, hi)):
            row, col = Bm[:, t].repeat_interleave(hpg, 1)[:, :, None, :], Cm[:, t].repeat_interleave(hpg, 1)[:, :, None, :]
            G1 = G1 + dy[:, t][..., None] * col
            d_C[:, t] = (h * dy[:, t][..., None]).sum(2).reshape(b, G, hpg, N).sum(2)
            gx = (G1 * x[:, t][..., None]).sum(2)
            d_B[:, t] = (gx * dt[:, t][..., None]).reshape(b, G, hpg, N).sum(2)
            gb = (G1 * row).sum(-1)
            d_X[:, t] = dt[:, t][..., None] * gb + st["D"].double()[:, None] * dy[:, t]
            decay = torch.exp(A * dt[:, t])
            G1 = decay[..., None, None] * G1
            da = (G1 * before[t - lo]).sum((-1, -2))
            d_dt[:, t] = (gb * x[:, t]).sum(-1) + A * da
            d_A += (dt[:, t] * da).sum(0)
            h = before[t - lo]
    d_dt = d_dt * torch.sigmoid(raw) * ((soft >= DT_MIN) & (soft <= DT_MAX))
    return dict(d_X=d_X, d_B=d_B, d_C=d_C, d_dt=d_dt, d_dt_bias=d_dt.sum((0, 1)), d_A_log=A * d_A,
                d_D=(x * dy).sum((0, 1, 3)), d_state0=G1)
