"""What the sequence-policy operators (serl_amd.sequence) are measured on: the gated recurrence, the root-mean-square norm
and the distillation loss, each in a plain form of elementary torch operations and as the library's own calls.

`own` selects the side: False = the plain form, True = the library."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
E4M3_MAX = 448.0            # largest finite value of torch.float8_e4m3fn
MAX_SCAN = 8 * 4096 * 2048      # elements of the largest listed case of each operator
MAX_NORM = 16384 * 4096
MAX_DISTILL = 2048 * 131072


# ------------------------------------------------------------------------------------------------------------ cases
def _scan(name, what, dtype, B, T, D, h0=False, starts=False, lengths=False, views=False):
    return dict(name=name, op="scan", what=what, dtype=dtype, B=B, T=T, D=D, h0=h0, starts=starts, lengths=lengths, views=views)


def _norm(name, what, dtype, R, N, residual=True, stream="same"):
    return dict(name=name, op="norm", what=what, dtype=dtype, R=R, N=N, residual=residual, stream=stream)


def _distill(name, dtype, R, V, K, tau=1.0, grad=True, coef=True, absent=0.0):
    return dict(name=name, op="distill", dtype=dtype, R=R, V=V, K=K, tau=tau, grad=grad, coef=coef, absent=absent)


def listed():
    return [
        # acting: one step of 64 environments, the state kept between calls; pure latency
        _scan("scan_step_64x1024", "step", "bf16", 64, 1, 1024, h0=True, starts=True),
        # a replay batch of 256 windows of 50 steps with episode borders inside, evaluated for its targets; gate and
        # candidate are the two halves of one projection
        _scan("scan_fwd_256x50x512", "fwd", "fp32", 256, 50, 512, h0=True, starts=True, views=True),
        # one very long episode (30 011 steps) through a trained memory: the time axis itself has to be split
        _scan("scan_fwd_1x30011x1024", "fwd", "bf16", 1, 30011, 1024, h0=True),
        # ragged demonstrations of an odd width (no wide loads), both directions
        _scan("scan_train_12x777x333", "train", "fp32", 12, 777, 333, starts=True, lengths=True),
        # the ordinary large training step: 8 sequences of 4096 steps, 2048 channels, both directions
        _scan("scan_train_8x4096x2048", "train", "bf16", 8, 4096, 2048, h0=True, starts=True),
        # serving: the norm before an 8-bit product, one token of 64 sequences; latency
        _norm("norm_fp8_64x4096", "fp8", "bf16", 64, 4096),
        # training at an odd width
        _norm("norm_train_5000x1001", "train", "fp32", 5000, 1001),
        # the ordinary training step over a batch of sequences
        _norm("norm_train_16384x4096", "train", "bf16", 16384, 4096),
        # a small discrete head: 256 rows of 256 action bins, teacher's 8 best; latency
        _distill("distill_256x256", "fp32", 256, 256, 8, tau=2.0),
        # few rows of a large vocabulary: a row has to be shared by several workgroups
        _distill("distill_16x131072", "bf16", 16, 131072, 100),
        # an odd vocabulary, rows that start at any alignment, teacher rows of unequal length
        _distill("distill_1500x50021", "bf16", 1500, 50021, 64, tau=1.5, absent=0.1),
        # the large training step
        _distill("distill_2048x131072", "bf16", 2048, 131072, 128),
    ]


def _spread(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi], odd ones and round ones."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.4 and v >= 16:
        step = 1 << max(3, v.bit_length() - 3)
        v = max(step, v // step * step)
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["scan", "scan", "norm", "norm", "distill", "distill"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "scan":
        what = rng.choice(["step", "fwd", "train", "train"])
        B, D = _spread(rng, 1, 256), _spread(rng, 16, 4096)
        T = 1 if what == "step" else _spread(rng, 1, 32768)
        most = MAX_SCAN // (2 if dtype == "fp32" else 1)
        while B * T * D > most:
            if B > 1:
                B = max(1, B // 2)
            else:
                T = max(1, T // 2)
        return dict(op="scan", what=what, dtype=dtype, B=B, T=T, D=D, h0=what == "step" or rng.random() < 0.5,
                    starts=rng.random() < 0.5, lengths=what != "step" and rng.random() < 0.4,
                    views=what != "step" and rng.random() < 0.4)
    if op == "norm":
        what = rng.choice(["fp8", "fwd", "train", "train"])
        R, N = _spread(rng, 1, 32768), _spread(rng, 64, 16384)
        most = MAX_NORM // (2 if dtype == "fp32" else 1)
        while R * N > most:
            R = max(1, R // 2)
        return dict(op="norm", what=what, dtype=dtype, R=R, N=N, residual=rng.random() < 0.7,
                    stream=rng.choice(["same", "same", "fp32"]))
    R, V = _spread(rng, 1, 8192), _spread(rng, 16, 200000)
    most = MAX_DISTILL // (2 if dtype == "fp32" else 1)
    while R * V > most:
        R = max(1, R // 2)
    return dict(op="distill", dtype=dtype, R=R, V=V, K=min(V, _spread(rng, 1, 256)), tau=rng.choice([1.0, 1.0, 0.5, 2.0, 3.7]),
                grad=rng.random() < 0.8, coef=rng.random() < 0.6, absent=rng.choice([0.0, 0.0, 0.2, 0.9]))


# ----------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, scale=1.0, shift=0.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).add_(shift).to(dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    s = {"case": case}
    if case["op"] == "scan":
        B, T, D = case["B"], case["T"], case["D"]
        # gates of a trained memory: from forgetting at once to remembering for hundreds of steps, by channel
        speed = normal(D, dtype=torch.float32, scale=2.0, shift=2.0)
        if case["views"]:
            both = torch.empty((B, T, 2 * D), device="cuda", dtype=dt)
            both[..., :D] = normal(B, T, D, dtype=torch.float32) + speed
            both[..., D:] = normal(B, T, D)
            s["gate"], s["x"] = both[..., :D], both[..., D:]
        else:
            s["gate"] = (normal(B, T, D, dtype=torch.float32) + speed).to(dt)
            s["x"] = normal(B, T, D)
        s["h0"] = normal(B, D, dtype=torch.float32) if case["h0"] else None
        s["starts"] = uniform(B, T) < 1.0 / 100 if case["starts"] else None
        s["lengths"] = (1 + uniform(B) * T).to(torch.int32).clamp_(max=T) if case["lengths"] else None
        if case["what"] == "step":
            s["gate"], s["x"] = s["gate"][:, 0], s["x"][:, 0]
            s["starts"] = s["starts"][:, 0].contiguous() if case["starts"] else None
        if case["what"] == "train":
            s["dy"] = normal(B, T, D)
            s["dh_last"] = normal(B, D, dtype=torch.float32)
    elif case["op"] == "norm":
        R, N = case["R"], case["N"]
        st = torch.float32 if case["stream"] == "fp32" else dt
        s["x"] = normal(R, N)
        s["residual"] = normal(R, N, dtype=st, scale=3.0) if case["residual"] else None
        s["weight"] = normal(N, scale=0.3, shift=1.0)
        if case["what"] == "train":
            s["dy"] = normal(R, N)
            s["ds"] = normal(R, N, dtype=st if case["residual"] else dt)
    else:
        R, V, K = case["R"], case["V"], case["K"]
        s["logits"] = normal(R, V, scale=2.5)
        s["index"] = _distinct(uniform(R, K), V, K)
        # the teacher agrees with the student on the order of things and is surer than it
        s["teacher"] = (normal(R, K, dtype=torch.float32, scale=2.0) + 6.0).to(dt)
        if case["absent"]:
            s["teacher"].masked_fill_(uniform(R, K) < case["absent"], -math.inf)
        s["coef"] = (uniform(R) + 0.5) / R * (uniform(R) < 0.9) if case["coef"] else None
    return s


def _distinct(u, V, K):
    """K different columns of [0, V) a row: one from each of K strips."""
    k = torch.arange(K, device=u.device)
    lo, hi = k * V // K, (k + 1) * V // K
    return torch.minimum(lo + (u * (hi - lo)).long(), hi - 1)


# --------------------------------------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if c["op"] == "scan":
        return _run_scan(s, c["what"])
    if c["op"] == "norm":
        return _run_norm(s, c["what"])
    return _run_distill(s, c)


def _run_scan(s, what):
    gate, x, h0, starts, lengths = s["gate"], s["x"], s["h0"], s["starts"], s["lengths"]
    if own:
        from serl_amd import sequence
        if what == "step":
            y, h_last = sequence.gated_scan_step(gate, x, h0, starts=starts)
            return {"y": y, "h_last": h_last}
        if what == "fwd":
            y, h_last = sequence.gated_scan(gate, x, h0=h0, starts=starts, lengths=lengths)
            return {"y": y, "h_last": h_last}
        y, h_last, saved = sequence.gated_scan(gate, x, h0=h0, starts=starts, lengths=lengths, save=True)
        dgate, dx, dh0 = sequence.gated_scan_backward(gate, x, saved, s["dy"], dh_last=s["dh_last"], starts=starts,
                                                      lengths=lengths)
        return {"y": y, "h_last": h_last, "dgate": dgate, "dx": dx, "dh0": dh0}
    if what == "step":
        f, b, _, _ = _gates(gate[:, None], x[:, None], None if starts is None else starts[:, None], None)
        h = f * h0[:, None] + b
        return {"y": h[:, 0].to(gate.dtype), "h_last": h[:, 0]}
    return _plain_scan(s, what)


def _gates(gate, x, starts, lengths):
    """Coefficients of h_t = keep_t h_{t-1} + b_t in 32 bits, the time mask and sigmoid(-gate)."""
    z = gate.float()
    rest = torch.sigmoid(-z)                # 1 - f without the cancellation
    keep, b = torch.sigmoid(z), rest * x.float()
    if starts is not None:
        keep = keep * (~starts)[..., None]
    live = None
    if lengths is not None:
        live = (torch.arange(z.shape[1], device=z.device) < lengths[:, None])[..., None]
        keep, b = torch.where(live, keep, 1.0), torch.where(live, b, 0.0)
    return keep, b, live, rest


def _doubling(a, b):
    """h_t = a_t h_{t-1} + b_t, h before the first = 0, along dim 1: spans of 1, 2, 4, ... steps joined with their left
    neighbours."""
    span = 1
    while span < a.shape[1]:
        b = torch.cat([b[:, :span], b[:, span:] + a[:, span:] * b[:, :-span]], 1)
        a = torch.cat([a[:, :span], a[:, span:] * a[:, :-span]], 1)
        span *= 2
    return b


def _plain_scan(s, what):
    gate, x, h0 = s["gate"], s["x"], s["h0"]
    dt = gate.dtype
    keep, b, live, rest = _gates(gate, x, s["starts"], s["lengths"])
    first = torch.zeros_like(b[:, 0]) if h0 is None else h0
    h = _doubling(keep, torch.cat([b[:, :1] + keep[:, :1] * first[:, None], b[:, 1:]], 1))
    out = {"y": (h if live is None else h * live).to(dt), "h_last": h[:, -1].contiguous()}
    if what == "fwd":
        return out
    before = torch.cat([first[:, None], h[:, :-1]], 1)
    del h, b
    if s["starts"] is not None:
        before = before * (~s["starts"])[..., None]
    dy = s["dy"].float()
    if live is not None:
        dy = dy * live
    dy = torch.cat([dy[:, :-1], dy[:, -1:] + s["dh_last"][:, None]], 1)
    # G_t = dy_t + keep_{t+1} G_{t+1}: the same recurrence with time turned round
    after = torch.cat([keep[:, 1:], torch.zeros_like(keep[:, :1])], 1)
    G = _doubling(after.flip(1), dy.flip(1)).flip(1)
    out["dh0"] = keep[:, 0] * G[:, 0]
    if live is not None:
        G = G * live
    out["dx"] = (G * rest).to(dt)
    out["dgate"] = (G * (before - x.float()) * rest * torch.sigmoid(gate.float())).to(dt)
    return out


def _run_norm(s, what):
    x, residual, w = s["x"], s["residual"], s["weight"]
    if own:
        from serl_amd import sequence
        if what == "fp8":
            q, scale, total = sequence.rms_norm_fp8(x, w, residual=residual)
            return {"q": q, "scale": scale, "sum": total}
        if what == "fwd":
            y, total = sequence.rms_norm(x, w, residual=residual)
            return {"y": y, "sum": total}
        y, total, rstd = sequence.rms_norm(x, w, residual=residual, save=True)
        dx, dw = sequence.rms_norm_backward(s["dy"], total, rstd, w, ds=s["ds"])
        return {"y": y, "sum": total, "dx": dx, "dweight": dw}
    # the norm is of the sum as it is stored: later layers and the backward pass see the same values
    total = x if residual is None else (x.float() + residual.float()).to(residual.dtype)
    v = total.float()
    rstd = torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6)
    if what == "fp8":
        y = v * rstd * w.float()
        top = y.abs().amax(-1)
        scale = torch.where(top > 0, (top / E4M3_MAX).clamp_min(2.0 ** -126), 1.0)
        return {"q": (y / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), "scale": scale, "sum": total}
    y = (v * rstd * w.float()).to(x.dtype)
    if what == "fwd":
        return {"y": y, "sum": total}
    dy = s["dy"].float()
    xh = v * rstd
    inner = dy * w.float()
    dx = rstd * (inner - xh * (inner * xh).mean(-1, keepdim=True)) + s["ds"].float()
    return {"y": y, "sum": total, "dx": dx.to(total.dtype), "dweight": (dy * xh).sum(0)}


def _run_distill(s, c):
    logits, teacher, index, coef, tau = s["logits"], s["teacher"], s["index"], s["coef"], c["tau"]
    if own:
        from serl_amd import sequence
        loss, d = sequence.topk_distill(logits, teacher, index, temperature=tau, coef=coef, grad=c["grad"])
        return {"loss": loss, "dlogits": d} if c["grad"] else {"loss": loss}
    t = teacher.float() / tau
    there = t > -math.inf
    top = t.amax(-1, keepdim=True)
    any_there = top > -math.inf
    e = torch.exp(t - torch.where(any_there, top, 0.0))
    total = e.sum(-1, keepdim=True)
    q = e / torch.where(any_there, total, 1.0)
    logq = t - torch.where(any_there, top + torch.log(total), 0.0)
    z = logits.float() / tau
    ztop = z.amax(-1, keepdim=True)
    lse = ztop + torch.log(torch.exp(z - ztop).sum(-1, keepdim=True))
    logp = z.gather(1, index) - lse
    factor = any_there[:, 0] * (1.0 if coef is None else coef)
    loss = factor * tau * tau * torch.where(there, q * (logq - logp), 0.0).sum(-1)
    if not c["grad"]:
        return {"loss": loss}
    d = torch.exp(z - lse).scatter_add(1, index, -q).mul_(factor[:, None] * tau)
    return {"loss": loss, "dlogits": d.to(logits.dtype)}


# ------------------------------------------------------------------------------------------- what a pass cannot spare
def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "scan":
        B, T, D = case["B"], case["T"], case["D"]
        n = B * T * D
        states = B * D * 4 * ((2 if case["h0"] else 1) + (2 if case["what"] == "train" else 0))
        mask = (B * T if case["starts"] else 0) + (4 * B if case["lengths"] else 0)
        # gate, x -> y; with the backward pass dy -> dgate, dx besides
        return {"bytes": n * e * (6 if case["what"] == "train" else 3) + states + mask,
                "flops": n * (25.0 if case["what"] == "train" else 9.0)}
    if case["op"] == "norm":
        R, N, what = case["R"], case["N"], case["what"]
        se = e if case["stream"] == "same" or not case["residual"] else 4
        read = R * N * (e + (se if case["residual"] else 0)) + N * e
        if what == "fp8":
            write = R * N * (1 + (se if case["residual"] else 0)) + 4 * R
        else:
            write = R * N * (e + (se if case["residual"] else 0))
        if what == "train":
            read += R * N * (e + se)
            write += R * N * se + 4 * N
        return {"bytes": read + write, "flops": R * N * (14.0 if what == "train" else 5.0)}
    R, V, K = case["R"], case["V"], case["K"]
    return {"bytes": R * V * e * (2 if case["grad"] else 1) + R * K * (8 + e) + R * (8 if case["coef"] else 4),
            "flops": R * V * (8.0 if case["grad"] else 4.0)}


# ------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "scan":
        return _exact_scan(s, case["what"])
    if case["op"] == "norm":
        return _exact_norm(s, case["what"])
    return _exact_distill(s, case)


def _exact_scan(s, what):
    """Step by step through time, as the recurrence is written."""
    gate, x = s["gate"].double(), s["x"].double()
    if what == "step":
        gate, x = gate[:, None], x[:, None]
    B, T, D = gate.shape
    starts = s["starts"]
    go = torch.ones((B, T, 1), dtype=torch.float64, device=x.device)
    if starts is not None:
        go = 1.0 - starts.reshape(B, T, 1).double()
    live = torch.ones((B, T, 1), dtype=torch.bool, device=x.device)
    if s["lengths"] is not None:
        live = torch.arange(T, device=x.device)[None, :, None] < s["lengths"][:, None, None]
    f = 1.0 / (1.0 + torch.exp(-gate))
    rest = 1.0 / (1.0 + torch.exp(gate))
    a = torch.where(live, f * go, 1.0)
    b = torch.where(live, rest * x, 0.0)
    h = torch.zeros((B, D), dtype=torch.float64, device=x.device) if s["h0"] is None else s["h0"].double()
    hs = torch.empty((T + 1, B, D), dtype=torch.float64, device=x.device)
    hs[0] = h
    a_t, b_t = a.unbind(1), b.unbind(1)
    for t in range(T):
        torch.addcmul(b_t[t], a_t[t], hs[t], out=hs[t + 1])
    hs = hs.transpose(0, 1)
    if what == "step":
        return {"y": hs[:, 1], "h_last": hs[:, 1]}
    out = {"y": torch.where(live, hs[:, 1:], 0.0), "h_last": hs[:, -1]}
    if what == "fwd":
        return out
    dy = torch.where(live, s["dy"].double(), 0.0).unbind(1)
    G = torch.empty((T, B, D), dtype=torch.float64, device=x.device)
    G[T - 1] = dy[T - 1] + s["dh_last"].double()
    for t in range(T - 2, -1, -1):
        torch.addcmul(dy[t], a_t[t + 1], G[t + 1], out=G[t])
    out["dh0"] = a_t[0] * G[0]
    G = torch.where(live, G.transpose(0, 1), 0.0)
    out["dx"] = G * rest
    out["dgate"] = G * (hs[:, :-1] * go - x) * f * rest
    return out


def _exact_norm(s, what):
    x, w = s["x"].double(), s["weight"].double()
    full = x if s["residual"] is None else x + s["residual"].double()
    v = full if s["residual"] is None else full.to(s["residual"].dtype).double()        # the stored sum is what is normed
    n = v.shape[1]
    size = torch.sqrt((v * v).sum(1, keepdim=True) / n + 1e-6)
    unit = v / size
    y = unit * w
    if what == "fp8":
        top = y.abs().max(1).values
        scale = torch.where(top > 0, torch.clamp(top / E4M3_MAX, min=2.0 ** -126), torch.ones_like(top))
        return {"q": y / scale[:, None], "scale": scale, "sum": full}
    if what == "fwd":
        return {"y": y, "sum": full}
    dy = s["dy"].double()
    inner = dy * w
    dx = (inner - unit * ((inner * unit).sum(1, keepdim=True) / n)) / size + s["ds"].double()
    return {"y": y, "sum": full, "dx": dx, "dweight": (dy * unit).sum(0)}


def _exact_distill(s, c):
    logits, tau = s["logits"], float(c["tau"])
    R, V = logits.shape
    losses, grads = [], []
    step = max(1, (1 << 26) // V)
    for r in range(0, R, step):
        rows = slice(r, r + step)
        z = logits[rows].double() / tau
        t = s["teacher"][rows].double() / tau
        dead = torch.isinf(t).all(1, keepdim=True)
        q = torch.softmax(torch.where(dead, 0.0, t), 1) * ~dead
        logp_all = torch.log_softmax(z, 1)
        logp = logp_all.gather(1, s["index"][rows])
        per = torch.special.xlogy(q, q) - torch.where(q > 0, q * logp, 0.0)
        c_r = 1.0 if s["coef"] is None else s["coef"][rows].double()
        c_r = c_r * (~dead[:, 0]).double()
        losses.append(c_r * tau * tau * per.sum(1))
        if c["grad"]:
            p = torch.exp(logp_all)
            p.scatter_add_(1, s["index"][rows], -q)
            grads.append(p * (c_r * tau)[:, None])
    out = {"loss": torch.cat(losses)}
    if c["grad"]:
        out["dlogits"] = torch.cat(grads)
    return out
