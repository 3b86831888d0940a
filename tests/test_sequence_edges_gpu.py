"""Edges of the operators of sequence policies (serl_amd/sequence.py): non-finite values, calls in place, strides and values at
the ends of their types, each against the operator's definition.  U, HALF and SMALL as in test_sequence_gpu.py."""
import math

import pytest
import torch

from test_sequence_gpu import DTYPES, HALF, SMALL, U, distill_reference, norm_inputs, scan_inputs, seq, within

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------- root-mean-square norm
@pytest.mark.parametrize("dtype,stream", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                          (torch.bfloat16, None)], ids=str)
def test_e4m3_codes_are_rounded_quotients(dev, dtype, stream):
    """The codes are those of y / scale, one correctly rounded division, to the bit: a product with 1 / scale has a rounding more and
    moves quotients next to the middle of two codes.  y = s rstd w has the same two roundings on the CPU."""
    s = seq()
    for R, N in ((64, 4096), (500, 2000), (3000, 200), (900, 1001), (20, 20000), (9, 5)):
        i = norm_inputs(dev, dtype, stream, R, N, R + N)
        _, total, rstd = s.rms_norm(i["x"], i["weight"], i["residual"], save=True)
        q, scale, total2 = s.rms_norm_fp8(i["x"], i["weight"], i["residual"])
        assert torch.equal(total, total2)
        y = total.float().cpu() * rstd.cpu()[:, None] * i["weight"].float().cpu()
        want = (y / scale.cpu()[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        assert torch.equal(scale.cpu(), y.abs().amax(1) / 448)
        off = int((q.cpu().view(torch.uint8) != want.view(torch.uint8)).sum())
        assert off == 0, f"{R} x {N}: {off} codes"
        if N > 5:                           # an infinite weight: the scale is infinite, what is finite is 0 of it, the rest NaN
            i["weight"][2] = math.inf
            q, scale, _ = s.rms_norm_fp8(i["x"], i["weight"], i["residual"])
            some = total[:, 2] != 0         # (0 inf = NaN: a row that holds a NaN has the scale NaN)
            assert bool((scale[some] == math.inf).all()) and bool(scale[~some].isnan().all()) and bool(q[:, 2].float().isnan().all())
            q = q.float()
            q[:, 2] = 0
            assert not q[some].any()


# ------------------------------------------------------------------------------- calls in place (raw pointers)
INPLACE = [(5, 5), (9, 61), (7, 130), (5, 520), (40, 777), (6, 2047), (3, 2048), (4, 4101), (3, 8193), (300, 9001), (6, 12289), (3, 16384),
           (4, 16385), (4, 16390), (600, 16390), (4, 16903), (4, 17409), (3, 20000), (3, 32761), (3, 32768)]


@pytest.mark.parametrize("dtype,stream", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)], ids=str)
def test_rms_norm_in_place(dev, dtype, stream):
    """y over x and the sum over the residual forward; dx over ds, or over the sum, backward: the bits of separate buffers."""
    from serl_amd import ops
    s = seq()
    code = {torch.float32: ops.F32, torch.bfloat16: ops.BF16, torch.float16: ops.F16}
    st = torch.cuda.current_stream(dev).cuda_stream
    for R, N in INPLACE:
        i = norm_inputs(dev, dtype, stream, R, N, N)
        w = i["weight"]
        y, total, rstd = s.rms_norm(i["x"], w, i["residual"], save=True)
        dx, dw = s.rms_norm_backward(i["dy"], total, rstd, w, i["ds"])
        x, res = i["x"].clone(), i["residual"].clone()
        ops.rms_norm_fwd(code[dtype], code[stream], code[dtype], R, N, x.data_ptr(), N, res.data_ptr(), N, w.data_ptr(), 1e-6, x.data_ptr(),
                         N, False, None, res.data_ptr(), N, None, st)
        assert torch.equal(x, y) and torch.equal(res, total), (R, N)
        q, scale, _ = s.rms_norm_fp8(i["x"], w, i["residual"])
        x, res, scale2 = i["x"].clone(), i["residual"].clone(), torch.empty(R, device=dev)
        e = x.element_size()                # the codes at the head of the row that they are made from
        ops.rms_norm_fwd(code[dtype], code[stream], code[dtype], R, N, x.data_ptr(), N, res.data_ptr(), N, w.data_ptr(), 1e-6, x.data_ptr(),
                         N * e, True, scale2.data_ptr(), res.data_ptr(), N, None, st)
        assert torch.equal(x.view(torch.uint8)[:, :N], q.view(torch.uint8)) and torch.equal(scale2, scale) and torch.equal(res, total), (R, N)
        n = ops.rms_norm_bwd_workspace_bytes(R, N)
        ws = torch.empty(max(1, n // 4), device=dev)
        dw2 = torch.empty(N, device=dev)
        for over in ("ds", "sum"):
            sm, ds = total.clone(), i["ds"].clone()
            out = ds if over == "ds" else sm
            ops.rms_norm_bwd(code[dtype], code[stream], code[dtype], R, N, i["dy"].data_ptr(), N, sm.data_ptr(), N, rstd.data_ptr(),
                             w.data_ptr(), ds.data_ptr(), N, out.data_ptr(), N, dw2.data_ptr(), ws.data_ptr(), n, st)
            assert torch.equal(out, dx) and torch.equal(dw2, dw), (R, N, over)


# ------------------------------------------------------------------------------------------------- gated recurrence
# every way through time: single steps in order, tiles of 16 to 128 steps, many tiles, a split time axis, narrow rows of each, groups of
# 8 and 16 threads, two workgroups per CU
SCAN_PLANS = [(2, 6, 24), (2, 6, 3), (2, 14, 24), (2, 30, 24), (2, 60, 24), (2, 120, 24), (2, 400, 72), (1, 3000, 72), (1, 3000, 24), (2, 2500, 90),
              (1, 3000, 3), (2, 500, 3), (20, 700, 512), (130, 300, 256), (300, 100, 130)]


def alike(got, want, keep, what):
    """The same bits wherever `keep` is."""
    assert torch.equal(got[keep], want[keep]), what


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,T,D", SCAN_PLANS)
@pytest.mark.parametrize("shift", [-5.0, 1.0], ids=["forgetting", "remembering"])
def test_what_is_not_finite_stays_until_an_episode_starts(dev, dtype, B, T, D, shift):
    """f is above 0 for every gate above -87, so a NaN or an infinity in h0, x, dy or dh_last reaches every step behind (before) it up to
    the next start, however small the product of the gates between; other channels, and steps it cannot reach, keep their bits."""
    s = seq()
    g = torch.Generator().manual_seed(T + D)
    r = lambda *n: torch.randn(n, generator=g)  # noqa: E731
    gate, x, dy = ((r(B, T, D) + c).to(dtype).to(dev) for c in (shift, 0, 0))
    h0, dh = r(B, D).to(dev), r(B, D).to(dev)
    stop = 4 * T // 5
    starts = torch.zeros((B, T), dtype=torch.bool, device=dev)
    starts[B - 1, stop] = True                       # the last sequence alone is cut
    b, c = B - 1, D // 2
    at = T // 4

    def both(x=x, h0=h0, dy=dy, dh=dh, st=None):
        y, h, saved = s.gated_scan(gate, x, h0, starts=st, save=True)
        return (y, h) + s.gated_scan_backward(gate, x, saved, dy, dh, starts=st)

    def put(t, *where, v=math.nan):
        t = t.clone()
        t[where] = v
        return t
    clean, cut = both(), both(st=starts)
    spots = torch.zeros((B, T, D), dtype=torch.bool, device=dev)
    state = torch.zeros((B, D), dtype=torch.bool, device=dev)
    state[b, c] = True

    def span(lo, hi):
        m = spots.clone()
        m[b, lo:hi, c] = True
        return m
    nothing = torch.zeros_like(state)
    for name, arg, st, ys, hs, dgs, dxs, d0s in (
            # what is NaN: y, h_last, dgate, dx, dh0
            ("x", dict(x=put(x, b, at, c)), None, span(at, T), state, span(at, T), span(0, 0), nothing),
            ("h0", dict(h0=put(h0, b, c)), None, span(0, T), state, span(0, T), span(0, 0), nothing),
            ("dy", dict(dy=put(dy, b, T - 1 - at, c)), None, span(0, 0), nothing, span(0, T - at), span(0, T - at), state),
            ("dh_last", dict(dh=put(dh, b, c)), None, span(0, 0), nothing, span(0, T), span(0, T), state),
            ("x, cut", dict(x=put(x, b, at, c)), starts, span(at, stop), nothing, span(at, stop), span(0, 0), nothing),
            ("h0, cut", dict(h0=put(h0, b, c)), starts, span(0, stop), nothing, span(0, stop), span(0, 0), nothing),
            ("dy, cut", dict(dy=put(dy, b, T - 1, c)), starts, span(0, 0), nothing, span(stop, T), span(stop, T), nothing),
            ("dh_last, cut", dict(dh=put(dh, b, c)), starts, span(0, 0), nothing, span(stop, T), span(stop, T), nothing)):
        got, want = both(**arg, st=st), clean if st is None else cut
        for out, u, v, nan in zip(("y", "h_last", "dgate", "dx", "dh0"), got, want, (ys, hs, dgs, dxs, d0s)):
            assert bool(u[nan].isnan().all()), f"{name} in {out}: {int((~u[nan].isnan()).sum())} of {int(nan.sum())} finite"
            alike(u, v, ~nan, f"{name} in {out}")
    y, h, *_ = both(h0=put(h0, b, c, v=-math.inf))
    assert bool((y[b, :, c] == -math.inf).all()) and float(h[b, c]) == -math.inf
    y, h, *_ = both(x=put(x, b, at, c, v=math.inf))
    assert bool((y[b, at:, c] == math.inf).all()) and float(h[b, c]) == math.inf
    *_, dx, d0 = both(dh=put(dh, b, c, v=math.inf))
    assert bool((dx[b, :, c] == math.inf).all()) and float(d0[b, c]) == math.inf
    *_, dx, d0 = both(dy=put(dy, b, T - 1 - at, c, v=-math.inf))
    assert bool((dx[b, :T - at, c] == -math.inf).all()) and float(d0[b, c]) == -math.inf
    alike(dx, clean[3], ~span(0, T - at), "dx")


@pytest.mark.parametrize("T", [6, 100, 3000])
def test_gates_of_zero_do_not_hide_a_nan(dev, T):
    """Where f itself is 0 in 32 bits, f h is still NaN for a NaN h."""
    s = seq()
    gate = torch.full((1, T, 40), -200.0, device=dev)
    x, h0 = torch.ones_like(gate), torch.zeros(1, 40, device=dev)
    h0[0, 7] = math.nan
    y, h = s.gated_scan(gate, x, h0)
    assert bool(y[0, :, 7].isnan().all()) and bool(h[0, 7].isnan())
    y[0, :, 7] = h[0, 7] = 1
    assert bool((y == 1).all()) and bool((h == 1).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,T,D", [(2, 6, 16), (2, 70, 16), (3, 200, 40), (1, 1500, 24), (2, 90, 3)])
def test_gate_gradient_at_a_start_keeps_small_gates(dev, dtype, B, T, D):
    """At an episode's first step dgate = -G x f (1 - f), to the relative accuracy of f: gates far below 0 too."""
    s = seq()
    i = scan_inputs(dev, dtype, B, T, D, T, h0=True)
    starts = torch.zeros((B, T), dtype=torch.bool, device=dev)
    starts[:, ::5] = True
    gate = i["gate"].clone()
    gate[:, ::5] = torch.tensor([-10.0, -17.0, -30.0, -60.0, 4.0], device=dev).to(dtype)[torch.arange(D, device=dev) % 5]
    _, _, saved = s.gated_scan(gate, i["x"], i["h0"], starts=starts, save=True)
    dgate, _, _ = s.gated_scan_backward(gate, i["x"], saved, i["dy"], i["dh_last"], starts=starts)
    z, x, dy = (t.double().cpu() for t in (gate, i["x"], i["dy"]))
    keep = torch.sigmoid(z) * ~starts.cpu()[..., None]
    f, rest = torch.sigmoid(z), torch.sigmoid(-z)
    C = i["dh_last"].double().cpu()
    size, want, tol = C.abs(), torch.zeros_like(z), torch.zeros_like(z)
    for t in range(T - 1, -1, -1):
        G, big = dy[:, t] + C, dy[:, t].abs() + size
        want[:, t] = -G * x[:, t] * f[:, t] * rest[:, t]
        # f and 1 - f: the exponent's |z| roundings and 4 more each, 3 products; G: at most 5 steps back to the next start, each with f's
        # roundings, a product and a sum, and the joins of threads, waves and tiles on the way (2 each, 16 at most), of the sum's size
        tol[:, t] = ((2 * z[:, t].abs() + 11) * G.abs() + (5 * (4 + 4 + 2) + 32) * big) * U * (x[:, t] * f[:, t] * rest[:, t]).abs()
        C, size = keep[:, t] * G, keep[:, t] * big
    at = starts.cpu()[..., None].expand(B, T, D)
    # a stored value's own rounding, or half a step among the type's smallest numbers
    least = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: SMALL}[dtype]
    within(dgate.cpu()[at], want[at], (tol + HALF[dtype] * want.abs() + least)[at], "dgate")


# --------------------------------------------------------------------------------------- the recurrence, element by element
def running(i):
    """The recurrence and its gradients in 64 bits, with what a count of roundings makes of each element: (values, bounds)."""
    z, x, dy = (i[k].double().cpu() for k in ("gate", "x", "dy"))
    B, T, D = z.shape
    live = torch.ones((B, T, 1), dtype=torch.bool)
    if i["lengths"] is not None:
        live = (torch.arange(T)[None] < i["lengths"].cpu().long()[:, None])[..., None]
    go = torch.ones((B, T, 1), dtype=torch.float64)
    if i["starts"] is not None:
        go = (~i["starts"].cpu())[..., None].double()
    f, rest = torch.sigmoid(z), torch.sigmoid(-z)
    # per step: f or 1 - f (its exponent's |z| roundings and 4 more), the product and the sum; 2 more for the joins that a tile hands on to
    # the next one, 40 roundings in 64 steps or more
    c = (z.abs() + 8) * U
    h = torch.zeros((B, D), dtype=torch.float64) if i["h0"] is None else i["h0"].double().cpu()
    size, err = h.abs(), torch.zeros_like(h)
    out, tol = {}, {}
    ys, ye, hs, he = [], [], [], []
    for t in range(T):
        k = f[:, t] * go[:, t]
        hs.append(h * go[:, t])
        # the tree of joins a state comes through: 4 levels in a wave, 16 waves, 2 roundings each
        he.append((err + 40 * U * size) * go[:, t])
        n, m = k * h + rest[:, t] * x[:, t], k * size + rest[:, t] * x[:, t].abs()
        e = k * err + c[:, t] * m
        h, size, err = (torch.where(live[:, t], u, v) for u, v in ((n, h), (m, size), (e, err)))
        ys.append(torch.where(live[:, t], h, torch.zeros_like(h)))
        ye.append(err + 40 * U * size)
    out["y"], tol["y"] = torch.stack(ys, 1), torch.stack(ye, 1)
    out["h_last"], tol["h_last"] = h, err + 40 * U * size
    C = i["dh_last"].double().cpu()
    size, err = C.abs(), torch.zeros_like(C)
    dg, dge, dx, dxe = ([None] * T for _ in range(4))
    for t in range(T - 1, -1, -1):
        lv = live[:, t]
        G, m, e = dy[:, t] + C, dy[:, t].abs() + size, err + U * (dy[:, t].abs() + size)
        eg = e + 40 * U * m
        ff, w = f[:, t] * rest[:, t], hs[t] - x[:, t]
        we = he[t] + U * (hs[t].abs() + x[:, t].abs())
        dg[t] = torch.where(lv, G * w * ff, torch.zeros_like(G))
        dge[t] = (eg * (w.abs() + we) + G.abs() * we + (2 * z[:, t].abs() + 12) * U * (G * w).abs()) * ff
        dx[t] = torch.where(lv, G * rest[:, t], torch.zeros_like(G))
        dxe[t] = (eg + (z[:, t].abs() + 6) * U * G.abs()) * rest[:, t]
        k = f[:, t] * go[:, t]
        C, size, err = (torch.where(lv, u, v) for u, v in ((k * G, C), (k * m, size), (k * e + c[:, t] * k * m, err)))
    for name, v, e in (("dgate", dg, dge), ("dx", dx, dxe)):
        out[name], tol[name] = torch.stack(v, 1), torch.stack(e, 1)
    out["dh0"], tol["dh0"] = C, err + 40 * U * size
    return out, tol


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,T,D", [(2, 5, 7), (2, 8, 64), (2, 14, 24), (3, 31, 24), (2, 60, 40), (2, 129, 33), (3, 257, 96), (1, 1100, 8),
                                   (2, 1537, 19), (2, 300, 3), (2, 900, 3), (40, 650, 256), (300, 100, 130)])
def test_gated_scan_within_the_roundings_of_each_element(dev, dtype, B, T, D):
    """Bounds that follow each element's own size, where those of test_gated_scan_matches_the_recurrence take the largest."""
    s = seq()
    for k, opt in enumerate(({}, {"starts": True}, {"starts": True, "lengths": True})):
        i = scan_inputs(dev, dtype, B, T, D, 7 * k + T + D, **opt)
        want, tol = running(i)
        y, h, saved = s.gated_scan(i["gate"], i["x"], i["h0"], i["starts"], i["lengths"], save=True)
        dg, dx, d0 = s.gated_scan_backward(i["gate"], i["x"], saved, i["dy"], i["dh_last"], i["starts"], i["lengths"])
        least = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: SMALL}[dtype]
        for name, got in (("y", y), ("h_last", h), ("dgate", dg), ("dx", dx), ("dh0", d0)):
            stored = HALF[dtype] * want[name].abs() + least if got.dtype == dtype and dtype != torch.float32 else 2.0 ** -149
            within(got, want[name], tol[name] * (1 + 2.0 ** -6) + stored, name)


# -------------------------------------------------------------------------------------------- top-logit distillation
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("tau", [0.5, 2.0 ** -20, 1.0, 3.0])
@pytest.mark.parametrize("R,V,K", [(6, 300, 6), (6, 12, 6), (6, 3000, 100), (6, 9001, 7), (150, 20000, 130), (6, 170000, 9)])
def test_teachers_at_the_ends_of_their_type(dev, dtype, tau, R, V, K):
    """Differences of a teacher's logits count, whatever their size over the temperature: slots that all hold the type's lowest (or the
    same largest) value weigh the same, one above the others' lowest takes everything."""
    s = seq()
    low, top = torch.finfo(dtype).min, torch.finfo(dtype).max
    g = torch.Generator().manual_seed(V)
    # a student whose columns lie within 4 tau of each other
    logits = (torch.rand((R, V), generator=g) * 4 * tau).to(dtype).to(dev)
    index = torch.stack([torch.randperm(V, generator=g)[:K] if K <= V else torch.arange(K) for _ in range(R)]).to(dev)
    teacher = torch.zeros((R, K), dtype=dtype, device=dev)
    q = torch.full((R, K), 1 / K, dtype=torch.float64)
    teacher[0] = low
    teacher[1] = top
    teacher[2] = low
    teacher[2, K - 1] = 0
    q[2] = 0
    q[2, K - 1] = 1
    teacher[3] = 1e30
    teacher[4] = low
    teacher[4, 1] = top
    q[4] = 0
    q[4, 1] = 1
    teacher[5] = low
    teacher[5, ::2] = -math.inf
    q[5] = 0
    q[5, 1::2] = 1 / len(range(1, K, 2))
    loss, d = s.topk_distill(logits, teacher, index, temperature=tau)
    logp = torch.log_softmax(logits.double().cpu() / tau, 1)
    want = tau * torch.exp(logp).scatter_add(1, index.cpu(), -q)
    # p and q <= 1: exponents of at most 4 with 3 roundings each, sums of up to 100 in a row (as check_distill), 1 for the difference
    n = (3 * 4 + 120) * U
    within(d, want, tau * n * (torch.exp(logp) + torch.zeros_like(logp).scatter_add(1, index.cpu(), q)) + HALF[dtype] * want.abs(), "dlogits")
    lp = logp.gather(1, index.cpu())
    rl = tau * tau * (torch.special.xlogy(q, q) - q * lp).sum(1)
    # log q, log p of at most 5 + log V <= 18, summed over at most 130 slots
    within(loss, rl, tau * tau * (n + (K + 20) * U) * 18, "loss")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tau", [0.25, 1.0, 2.0])
@pytest.mark.parametrize("R,V,K", [(4, 300, 6), (4, 12, 6), (4, 3000, 100), (150, 20000, 70), (4, 170000, 9)])
def test_loss_of_a_column_that_holds_the_lowest_value(dev, dtype, tau, R, V, K):
    """A student's column at the type's lowest value is masked, not impossible: tau q |low| is the loss, finite where the type of the
    sum holds it."""
    s = seq()
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(V)
    logits = torch.randn((R, V), generator=g).to(dtype).to(dev)
    index = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(R)]).to(dev)
    teacher = torch.randn((R, K), generator=g).to(dtype).to(dev)
    logits[0, index[0, 2]] = low
    logits[1, index[1, :3]] = low
    coef = torch.full((R,), 0.25, device=dev)
    i = dict(logits=logits, teacher=teacher, index=index, coef=coef)
    rl, _, q, lp, _ = distill_reference(i, tau)
    loss, d = s.topk_distill(logits, teacher, index, temperature=tau, coef=coef)
    assert bool((rl[:2] > 0.2 * tau * -low * q.gather(1, torch.full((R, 1), 2))[:2, 0]).all()) and bool(d.isfinite().all())
    # the terms are all above 0 but for log q: q's roundings (exponents of at most 12 / tau, K slots), those of log p (200 as for the
    # gradient, its own and the products)
    size = 0.25 * tau * tau * (q * (torch.log(q.clamp_min(1e-300)).abs() + lp.abs())).sum(1)
    within(loss, rl, (3 * 12 / tau + K + 230) * U * size, "loss")


# ------------------------------------------------------------------------------------------------- short windows
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("T", [2, 3, 5, 8])
def test_short_windows_whose_steps_lie_far_apart(dev, dtype, T):
    """Up to 8 steps a tensor's rows may be any distance apart, backward as forward: time-major batches, 2^29 bytes and more a step.
    The gaps stay as they were."""
    s = seq()
    B, D = 3, 24
    e = 4 if dtype == torch.float32 else 2
    far = (1 << 30) // e if T <= 5 else (1 << 29) // e          # (T - 1) steps: 2^30 .. 2^32 bytes
    i = scan_inputs(dev, dtype, B, T, D, T, starts=True, lengths=True)
    store = torch.zeros((T - 1) * far + 5 * B * D, dtype=dtype, device=dev)
    view = lambda k: torch.as_strided(store, (B, T, D), (D, far, 1), k * B * D)  # noqa: E731
    gate, x, dy, dgate, dx = (view(k) for k in range(5))
    gate.copy_(i["gate"])
    x.copy_(i["x"])
    dy.copy_(i["dy"])
    opt = dict(starts=i["starts"], lengths=i["lengths"])
    want = s.gated_scan(i["gate"], i["x"], i["h0"], save=True, **opt)
    got = s.gated_scan(gate, x, i["h0"], save=True, **opt)
    assert all(torch.equal(u, v) for u, v in zip(got, want))
    wg = s.gated_scan_backward(i["gate"], i["x"], want[2], i["dy"], i["dh_last"], **opt)
    gg = s.gated_scan_backward(gate, x, want[2], dy, i["dh_last"], out=(dgate, dx), **opt)
    assert gg[0] is dgate and gg[1] is dx
    # threads join in another order than with near rows: 8 steps of at most 10 roundings each, |G| <= 9 * 5, |h| + |x| <= 10
    tol = 8 * 10 * U * 45
    for k, (u, v) in enumerate(zip(gg, wg)):
        within(u, v, 2 * ((tol * 10 / 4 if k == 0 else tol) + HALF[dtype] * v.double().abs().cpu() + SMALL), "far steps")
    again = s.gated_scan_backward(gate, x, want[2], dy, i["dh_last"], **opt)
    assert all(torch.equal(u, v) for u, v in zip(again, gg))
    assert torch.equal(gate, i["gate"]) and torch.equal(x, i["x"]) and torch.equal(dy, i["dy"])
    inner = store.clone()
    for k in range(5):
        torch.as_strided(inner, (B, T, D), (D, far, 1), k * B * D).zero_()
    assert not inner.any()


@pytest.mark.parametrize("T", [6, 100, 3000])
def test_gates_of_zero_forget_the_largest_states(dev, T):
    """What is left of a state of fp32's largest size behind gates that are 0, or whose product is, is below 1e-6."""
    s = seq()
    for dtype in DTYPES:
        for low, at in ((-math.inf, 0), (-200.0, 0), (-80.0, 2), (-20.0, 5)):      # f^at h0 is below 1e-6, and behind it the x of the last steps
            gate = torch.full((2, T, 40), low, dtype=dtype, device=dev)
            x, h0 = torch.full_like(gate, 0.5), torch.full((2, 40), 3e38, device=dev)
            y, h, saved = s.gated_scan(gate, x, h0, save=True)
            within(y[:, at:], torch.full((2, T - at, 40), 0.5), 2.0 ** -20 + HALF[dtype], "y")
            within(h, torch.full((2, 40), 0.5), 2.0 ** -20, "h_last")
            _, _, d0 = s.gated_scan_backward(gate, x, saved, x, torch.full_like(h0, 3e38))
            # dh0 = sum of f^(t+1) dy_t + f^T dh_last
            f = 1 / (1 + math.exp(min(700.0, -low)))
            want = 0.5 * f / (1 - f) + (3e38 * f ** T if f ** T > 1e-60 else 0)
            within(d0, torch.full((2, 40), want), 2.0 ** -20 + abs(want) * T * 60 * U, "dh0")
