"""The operators of sequence policies (serl_amd/sequence.py) against plain 64-bit statements of the same formulas.

Tolerances.  A stored value carries one rounding, half a step: HALF[dtype] of its size.  What is computed in 32 bits before
it is bounded by counting roundings of 2^-24 (U below); the counts stand beside the checks."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {d: torch.finfo(d).eps / 2 for d in DTYPES}
U = 2.0 ** -24
SMALL = 2.0 ** -25      # half a step among fp16's subnormal numbers: they are multiples of 2^-24 (smallest_normal 2^-14 * eps 2^-10)


def seq():
    from serl_amd import sequence
    return sequence


def within(got, ref, tol, what):
    """|got - ref| <= tol element by element (tol: a number or a tensor like ref); ref finite."""
    got = got.detach().double().cpu()
    ref = ref.detach().double().cpu()
    tol = torch.as_tensor(tol, dtype=torch.float64)
    if not ref.numel():
        assert got.shape == ref.shape, what
        return
    bad = ~((got - ref).abs() <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - ref).abs().nan_to_num(math.inf).max()):.3e}, tolerance {float(tol.max()):.3e}"


# ------------------------------------------------------------------------------------------------- gated recurrence
def scan_inputs(dev, dtype, B, T, D, seed, h0=True, starts=False, lengths=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    gate = (r(B, T, D) * 2 + 1).clamp_(-6, 4).to(dtype)      # f <= sigmoid(4) = 0.982: a memory of 56 steps
    x, dy = r(B, T, D).to(dtype), r(B, T, D).to(dtype)
    out = dict(gate=gate, x=x, dy=dy, dh_last=r(B, D), h0=r(B, D) if h0 else None, starts=None, lengths=None)
    if starts:
        out["starts"] = torch.rand((B, T), generator=g) < 0.15
        out["starts"][0, :2] = True
    if lengths:
        out["lengths"] = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
        out["lengths"][0] = T
        out["lengths"][-1] = 0 if B > 1 else max(0, T - 1)
    return {k: None if v is None else v.to(dev) for k, v in out.items()}


def scan_reference(gate, x, h0, starts, lengths, dy=None, dh_last=None):
    """The recurrence step by step in 64 bits, its gradients by autograd."""
    gate, x = (t.double().cpu().requires_grad_() for t in (gate, x))
    B, T, D = gate.shape
    first = torch.zeros((B, D), dtype=torch.float64) if h0 is None else h0.double().cpu()
    first.requires_grad_()
    h, ys = first, []
    f, xs = torch.sigmoid(gate).unbind(1), x.unbind(1)
    for t in range(T):
        prev = h if starts is None else torch.where(starts[:, t, None].cpu(), torch.zeros_like(h), h)
        new = f[t] * prev + (1 - f[t]) * xs[t]
        live = torch.ones((B, 1), dtype=torch.bool) if lengths is None else (t < lengths.cpu().long())[:, None]
        h = torch.where(live, new, h)
        ys.append(torch.where(live, new, torch.zeros_like(new)))
    y = torch.stack(ys, 1)
    if dy is None:
        return y, h
    total = (y * dy.double().cpu()).sum() + (h * dh_last.double().cpu()).sum()
    return (y, h) + torch.autograd.grad(total, (gate, x, first))


# 56 steps of memory, each with at most 6 roundings of the gate, the products and the joins of tiles
SCAN_STATE = 56 * 6 * U


def check_scan(i, dtype, with_backward=True):
    s = seq()
    y, h, saved = s.gated_scan(i["gate"], i["x"], h0=i["h0"], starts=i["starts"], lengths=i["lengths"], save=True)
    y2, h2 = s.gated_scan(i["gate"], i["x"], h0=i["h0"], starts=i["starts"], lengths=i["lengths"])
    assert torch.equal(y, y2) and torch.equal(h, h2) and y.dtype == dtype and h.dtype == torch.float32
    ry, rh, rg, rx, r0 = scan_reference(i["gate"], i["x"], i["h0"], i["starts"], i["lengths"], i["dy"], i["dh_last"])
    hm = max(1.0, float(rh.detach().abs().max()), float(ry.detach().abs().max()))
    within(y, ry, SCAN_STATE * hm + HALF[dtype] * ry.detach().abs() + SMALL, "y")
    within(h, rh, SCAN_STATE * hm, "h_last")
    if not with_backward:
        return
    dg, dx, d0 = s.gated_scan_backward(i["gate"], i["x"], saved, i["dy"], dh_last=i["dh_last"], starts=i["starts"],
                                       lengths=i["lengths"])
    # |G| is at most the sum of what reaches a step: bounded by (56 + 1) of the largest |dy|, |dh_last|
    gm = 57 * max(float(i["dy"].abs().max()), float(i["dh_last"].abs().max()))
    xm = float(i["x"].abs().max())
    within(d0, r0, SCAN_STATE * gm, "dh0")
    within(dx, rx, SCAN_STATE * gm + HALF[dtype] * rx.abs() + SMALL, "dx")
    # dgate = G (h - x) f (1 - f): the errors of G and of h, each by the other's size, with f (1 - f) <= 1/4; 2^-26: half
    # a step among fp16's smallest numbers
    within(dg, rg, 2 * SCAN_STATE * gm * (hm + xm) / 4 + HALF[dtype] * rg.abs() + SMALL, "dgate")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (3, 1, 64), (2, 5, 7), (4, 8, 64), (2, 9, 16), (1, 31, 24), (2, 127, 40), (1, 128, 136),
                                   (2, 129, 33), (3, 257, 96), (2, 385, 65), (1, 640, 12), (2, 641, 10), (34, 645, 256), (35, 643, 256),
                                   (1, 1100, 8), (2, 1537, 19), (1, 4700, 72), (3, 1030, 701), (2, 2433, 131), (2, 300, 3),
                                   (2, 900, 29), (3, 60, 80), (3, 200, 72), (2, 1500, 96), (150, 700, 90)])
def test_gated_scan_matches_the_recurrence(dev, dtype, B, T, D):
    for k, opt in enumerate(({}, {"starts": True}, {"lengths": True, "h0": False}, {"starts": True, "lengths": True})):
        check_scan(scan_inputs(dev, dtype, B, T, D, 100 * k + T + D, **opt), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_gated_scan_gradient_matches_differences(dev, dtype):
    """<gradient, direction> against the central difference of the kernel's own outputs (state only, so fp32)."""
    s = seq()
    B, T, D = 2, 150, 24
    i = scan_inputs(dev, torch.float32, B, T, D, 5, starts=True)
    y, h, saved = s.gated_scan(i["gate"], i["x"], h0=i["h0"], starts=i["starts"], save=True)
    dg, dx, d0 = s.gated_scan_backward(i["gate"], i["x"], saved, i["dy"], dh_last=i["dh_last"], starts=i["starts"])
    g = torch.Generator(device=dev).manual_seed(1)
    vg, vx, v0 = (torch.randn(t.shape, generator=g, device=dev) for t in (i["gate"], i["x"], i["h0"]))

    def value(e):
        y, h = s.gated_scan(i["gate"] + e * vg, i["x"] + e * vx, h0=i["h0"] + e * v0, starts=i["starts"])
        return float((y.double() * i["dy"]).sum() + (h.double() * i["dh_last"]).sum())
    e = 2.0 ** -9
    want = float((dg.double() * vg).sum() + (dx.double() * vx).sum() + (d0.double() * v0).sum())
    got = (value(e) - value(-e)) / (2 * e)
    # size of the value's terms sqrt(B T D) ~ 85, each off by SCAN_STATE, over 2 e; the cubic term e^2 / 6 of the same size times 57^2
    n = math.sqrt(B * T * D)
    assert abs(got - want) <= n * 4 * SCAN_STATE / (2 * e) + n * e * e / 6 * 57 ** 2, (got, want)


def test_gated_scan_step_equals_a_scan_of_one_step_and_may_run_in_place(dev):
    s = seq()
    for dtype in DTYPES:
        for B, D in ((1, 1), (3, 7), (64, 1024), (5, 40)):
            i = scan_inputs(dev, dtype, B, 6, D, B, starts=True)
            h = i["h0"].clone()
            y, h_last = s.gated_scan(i["gate"], i["x"], h0=i["h0"], starts=i["starts"])
            for t in range(6):
                before = h.clone()
                yt, new = s.gated_scan_step(i["gate"][:, t], i["x"][:, t], h, starts=i["starts"][:, t])
                assert torch.equal(h, before)
                ys, hs = s.gated_scan_step(i["gate"][:, t], i["x"][:, t], h, starts=i["starts"][:, t], h_out=h)
                assert hs is h and torch.equal(h, new) and torch.equal(yt, ys) and torch.equal(yt, y[:, t])
            assert torch.equal(h, h_last)


def test_gated_scan_takes_views_and_writes_views(dev):
    """gate and x as halves of one projection, gradients into the halves of one buffer, odd offsets, a batch stride of 0."""
    s = seq()
    for dtype in (torch.float32, torch.bfloat16):
        for D, off in ((64, 0), (64, 1), (33, 3)):
            i = scan_inputs(dev, dtype, 3, 140, D, D + off, starts=True, lengths=True)
            both = torch.full((3, 140, 2 * D + off + 5), float("nan"), dtype=dtype, device=dev)
            both[..., off:off + D], both[..., off + D:off + 2 * D] = i["gate"], i["x"]
            gate, x = both[..., off:off + D], both[..., off + D:off + 2 * D]
            a = s.gated_scan(i["gate"], i["x"], i["h0"], i["starts"], i["lengths"], save=True)
            b = s.gated_scan(gate, x, i["h0"], i["starts"], i["lengths"], save=True)
            grads = torch.full_like(both, 7.0)
            out = grads[..., off:off + D], grads[..., off + D:off + 2 * D]
            ga = s.gated_scan_backward(i["gate"], i["x"], a[2], i["dy"], i["dh_last"], i["starts"], i["lengths"])
            s.gated_scan_backward(gate, x, b[2], i["dy"], i["dh_last"], i["starts"], i["lengths"], out=out)
            tol = 2 * 60 * 6 * U * 57 * 6
            for u, v in zip(a[:2] + ga[:2], b[:2] + out):      # another order of joins than with wide loads
                within(v, u, tol + 2 * HALF[dtype] * u.double().abs().cpu(), "view")
            assert bool((grads[..., :off] == 7).all()) and bool((grads[..., off + 2 * D:] == 7).all())
    i = scan_inputs(dev, torch.float32, 1, 50, 16, 3)
    y, h = s.gated_scan(i["gate"].expand(4, 50, 16), i["x"].expand(4, 50, 16), h0=i["h0"].expand(4, 16))
    y1, h1 = s.gated_scan(i["gate"], i["x"], h0=i["h0"])
    assert torch.equal(y, y1.expand_as(y)) and torch.equal(h, h1.expand_as(h))
    # channels that are not contiguous are copied first
    y2, _ = s.gated_scan(i["gate"].transpose(1, 2).contiguous().transpose(1, 2), i["x"], h0=i["h0"])
    assert torch.equal(y2, y1)


@pytest.mark.parametrize("T", [6, 300, 2100])
def test_gated_scan_keeps_what_is_masked_out(dev, T):
    """NaN and infinities behind a sequence's length do nothing; those of an episode end with it."""
    s = seq()
    B, D = 3, 24
    for dtype in (torch.float32, torch.bfloat16):
        i = scan_inputs(dev, dtype, B, T, D, T)
        n = torch.tensor([0, T // 2, T - 1], dtype=torch.int32, device=dev)
        clean = s.gated_scan(i["gate"], i["x"], i["h0"], lengths=n, save=True)
        cg = s.gated_scan_backward(i["gate"], i["x"], clean[2], i["dy"], i["dh_last"], lengths=n)
        bad = {k: i[k].clone() for k in ("gate", "x", "dy")}
        for b in range(B):
            bad["gate"][b, int(n[b]):] = float("nan")
            bad["x"][b, int(n[b]):] = float("inf")
            bad["dy"][b, int(n[b]):] = float("nan")
        got = s.gated_scan(bad["gate"], bad["x"], i["h0"], lengths=n.long(), save=True)
        gg = s.gated_scan_backward(bad["gate"], bad["x"], got[2], bad["dy"], i["dh_last"], lengths=n)
        for u, v in zip(clean + cg, got + gg):
            assert torch.equal(u, v)
        for b in range(B):
            assert not got[0][b, int(n[b]):].any() and not gg[0][b, int(n[b]):].any() and not gg[1][b, int(n[b]):].any()
        assert torch.equal(got[1][0], i["h0"][0]) and torch.equal(gg[2][0], i["dh_last"][0])
        # an episode full of NaN between two clean ones
        lo, hi = T // 3, T // 2
        st = torch.zeros((B, T), dtype=torch.bool, device=dev)
        st[:, lo] = st[:, hi] = True
        clean = s.gated_scan(i["gate"], i["x"], i["h0"], starts=st, save=True)
        cg = s.gated_scan_backward(i["gate"], i["x"], clean[2], i["dy"], i["dh_last"], starts=st)
        bad = {k: i[k].clone() for k in ("gate", "x", "dy")}
        for k in bad:
            bad[k][:, lo:hi] = float("nan")
        got = s.gated_scan(bad["gate"], bad["x"], i["h0"], starts=st, save=True)
        gg = s.gated_scan_backward(bad["gate"], bad["x"], got[2], bad["dy"], i["dh_last"], starts=st)
        for u, v in zip(clean[:1] + cg[:2], got[:1] + gg[:2]):
            assert torch.equal(u[:, :lo], v[:, :lo]) and torch.equal(u[:, hi:], v[:, hi:])
            assert bool(v[:, lo:hi].isnan().all())
        assert torch.equal(clean[1], got[1]) and torch.equal(cg[2], gg[2])


def test_gated_scan_extreme_gates(dev):
    """Gates at the ends of the type: remember exactly, replace exactly, infinities included."""
    s = seq()
    for dtype in DTYPES:
        big = torch.finfo(dtype).max
        gate = torch.tensor([big, float("inf"), -big, float("-inf"), 200.0, -200.0], dtype=dtype, device=dev).repeat(2, 40, 4)
        x = torch.randn((2, 40, 24), device=dev).to(dtype)
        h0 = torch.randn((2, 24), device=dev)
        y, h, saved = s.gated_scan(gate, x, h0=h0, save=True)
        keep = gate[0, 0] > 0
        assert torch.equal(h[:, keep], h0[:, keep]) and torch.equal(y[:, :, ~keep], x[:, :, ~keep])
        dg, dx, d0 = s.gated_scan_backward(gate, x, saved, torch.ones_like(x))
        assert not dg.any() and not dx[:, :, keep].any() and bool((dx[:, :, ~keep] == 1).all())
        assert bool((d0[:, keep] == 40).all()) and not d0[:, ~keep].any()


def test_gated_scan_empty_sizes(dev):
    s = seq()
    h0 = torch.randn((3, 8), device=dev)
    e = torch.empty((3, 0, 8), device=dev)
    y, h, saved = s.gated_scan(e, e, h0=h0, save=True)
    assert y.shape == (3, 0, 8) and torch.equal(h, h0) and saved.shape == (3, 0, 8)
    assert not s.gated_scan(e, e)[1].any()
    dg, dx, d0 = s.gated_scan_backward(e, e, saved, e, dh_last=h0)
    assert dg.shape == dx.shape == (3, 0, 8) and torch.equal(d0, h0)
    for shape in ((0, 5, 8), (2, 5, 0)):
        e = torch.empty(shape, device=dev)
        y, h, saved = s.gated_scan(e, e, save=True)
        assert y.shape == shape and h.shape == (shape[0], shape[2])
        assert s.gated_scan_backward(e, e, saved, e)[0].shape == shape


def test_gated_scan_offsets_beyond_32_bits(dev):
    """Steps that lie 2^26 elements apart: the last ones are beyond 2^32 bytes and 2^31 elements."""
    s = seq()
    T, D, far = 40, 16, 1 << 26
    store = torch.empty((T - 1) * far + 2 * D, dtype=torch.bfloat16, device=dev)
    gate, x = (torch.as_strided(store, (1, T, D), (0, far, 1), o) for o in (0, D))
    i = scan_inputs(dev, torch.bfloat16, 1, T, D, 9)
    gate.copy_(i["gate"])
    x.copy_(i["x"])
    a = s.gated_scan(i["gate"], i["x"], i["h0"], save=True)
    b = s.gated_scan(gate, x, i["h0"], save=True)
    ga = s.gated_scan_backward(i["gate"], i["x"], a[2], i["dy"], i["dh_last"])
    gb = s.gated_scan_backward(gate, x, b[2], i["dy"], i["dh_last"])
    # rows this far apart run the kernel of narrow loads, whose threads join in another order: both results are within
    # check_scan's tolerance of the recurrence, with |G| <= 57 max |dy| <= 57 * 5 and |h| + |x| <= 10
    for u, v in zip(a + ga, b + gb):
        within(v, u, 2 * (2 * SCAN_STATE * 57 * 5 * 10 / 4 + HALF[torch.bfloat16] * u.double().abs().cpu()), "far rows")


def replayed(dev, fn, outputs_of):
    """fn captured and replayed with eager work between the replays: every replay gives the eager call's bits."""
    want = [t.clone() for t in outputs_of(fn())]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = outputs_of(fn())
    for k in range(4):
        for t in out:
            t.zero_()
        eager = outputs_of(fn())
        graph.replay()
        torch.cuda.synchronize()
        for u, v, w in zip(out, eager, want):
            assert torch.equal(u, w) and torch.equal(v, w), f"replay {k}"


def test_gated_scan_in_graphs_and_on_other_streams(dev):
    s = seq()
    for T in (1, 60, 2000):
        i = scan_inputs(dev, torch.bfloat16, 2, T, 72, T, starts=True, lengths=True)

        def train():
            y, h, saved = s.gated_scan(i["gate"], i["x"], i["h0"], i["starts"], i["lengths"], save=True)
            return (y, h) + s.gated_scan_backward(i["gate"], i["x"], saved, i["dy"], i["dh_last"], i["starts"], i["lengths"])
        replayed(dev, train, list)
        want = train()
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            got = train()
        side.synchronize()
        for u, v in zip(want, got):
            assert torch.equal(u, v)


# ------------------------------------------------------------------------------------------- root-mean-square norm
def norm_inputs(dev, dtype, stream, R, N, seed, wtype=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    return dict(x=r(R, N).to(dtype).to(dev), residual=None if stream is None else (3 * r(R, N)).to(stream).to(dev),
                weight=(1 + 0.3 * r(N)).to(wtype or dtype).to(dev), dy=r(R, N).to(dtype).to(dev),
                ds=r(R, N).to(stream or dtype).to(dev))


# mean of squares: a thread adds at most 32 of them, 6 shuffle steps and 16 waves; half of that for the root, then the
# division, the root and the two products
NORM_Y = (54 / 2 + 6) * U


def check_norm(i, dtype, eps=1e-6):
    s = seq()
    R, N = i["x"].shape
    y, total, rstd = s.rms_norm(i["x"], i["weight"], residual=i["residual"], eps=eps, save=True)
    y2, total2 = s.rms_norm(i["x"], i["weight"], residual=i["residual"], eps=eps)
    assert torch.equal(y, y2) and torch.equal(total, total2) and y.dtype == dtype and rstd.dtype == torch.float32
    if i["residual"] is None:
        assert total is i["x"]
    else:
        full = i["x"].double() + i["residual"].double()
        assert total.dtype == i["residual"].dtype
        within(total, full, (HALF[total.dtype] + U) * full.abs().cpu() + SMALL, "sum")
    v, w = total.double().cpu(), i["weight"].double().cpu()
    r = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    ref = v * r * w
    within(rstd, r[:, 0], NORM_Y * r[:, 0], "rstd")
    within(y, ref, (NORM_Y + HALF[dtype]) * ref.abs() + SMALL, "y")
    q, scale, total3 = s.rms_norm_fp8(i["x"], i["weight"], residual=i["residual"], eps=eps)
    assert q.dtype == torch.float8_e4m3fn and torch.equal(total3, total)
    top = ref.abs().amax(1)
    within(scale, top / 448, (NORM_Y + 2 * U) * top / 448, "scale")
    # e4m3: half a step is 2^-4 of the value, or 2^-10 of the scale among its smallest numbers
    back = q.double().cpu() * scale.double().cpu()[:, None]
    within(back, ref, (2.0 ** -4 + 2 * NORM_Y + 4 * U) * ref.abs() + 2.0 ** -10 * scale.double().cpu()[:, None], "8 bits")
    for ds in (i["ds"], None):
        dx, dw = s.rms_norm_backward(i["dy"], total, rstd, i["weight"], ds=ds)
        assert dx.dtype == total.dtype and dw.dtype == torch.float32 and dw.shape == (N,)
        vv, ww = v.clone().requires_grad_(), w.clone().requires_grad_()
        out = vv / torch.sqrt((vv * vv).mean(1, keepdim=True) + eps) * ww
        rx, rw = torch.autograd.grad((out * i["dy"].double().cpu()).sum(), (vv, ww))
        add = 0 if ds is None else ds.double().cpu()
        dyw, xh = i["dy"].double().cpu() * w, v * r
        size = r * (dyw.abs() + xh.abs() * (dyw * xh).abs().mean(1, keepdim=True)) + (0 if ds is None else add.abs())
        within(dx, rx + add, 2 * (NORM_Y + 54 * U) * size + HALF[dx.dtype] * (rx + add).abs() + SMALL, "dx")
        # at least 512 shares (256 for R < 512), or one per row: a share adds up to R / 256 rows and four lanes; the last step's lanes
        # up to 16 shares, with more than 512 shares no more than R / 8 / 32; then 32 lanes
        within(dw, rw, (R / 128 + 52 + NORM_Y / U) * U * (i["dy"].double().cpu() * xh).abs().sum(0) + 1e-30, "dweight")


@pytest.mark.parametrize("dtype,stream", [(torch.float32, None), (torch.float32, torch.float32), (torch.bfloat16, None),
                                          (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                          (torch.float16, torch.float16), (torch.float16, torch.float32)], ids=str)
def test_rms_norm_matches_its_formulas(dev, dtype, stream):
    for R, N in ((1, 1), (3, 7), (70, 3), (3, 8), (4, 9), (5, 64), (1, 512), (6, 520), (2, 1000), (3, 1001), (2, 1024), (3, 2048),
                 (2, 2056), (5, 4096),
                 (2, 4097), (3, 8192), (1, 12288), (2, 16384), (1, 20000), (2, 32767), (1, 32768)):
        check_norm(norm_inputs(dev, dtype, stream, R, N, R + N), dtype)
    check_norm(norm_inputs(dev, dtype, stream, 3, 264, 1, wtype=torch.float32), dtype, eps=0.5)


@pytest.mark.parametrize("R,N", [(513, 40), (2051, 33), (700, 1100), (1030, 2064), (70001, 5), (33000, 128), (5001, 249), (9000, 333),
                                 (300, 9001)])
def test_rms_norm_many_rows(dev, R, N):
    for dtype in (torch.float32, torch.bfloat16):
        check_norm(norm_inputs(dev, dtype, dtype, R, N, R), dtype)


# rows that start at any element, NaN around them: each shape of the kernel with its last vector moved left
@pytest.mark.parametrize("dtype,stream", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)],
                         ids=str)
def test_rms_norm_rows_at_any_element(dev, dtype, stream):
    for R, N in ((9, 8), (7, 61), (5, 130), (6, 257), (3, 777), (2, 1030), (3, 2047), (2, 4101), (3, 8193), (2, 16390), (2, 32761)):
        i = norm_inputs(dev, dtype, stream, R, N, R * N)
        for off, pad in ((1, 2), (4, 4)):
            for k in ("x", "residual", "dy", "ds"):
                big = torch.full((R, off + N + pad), float("nan"), dtype=i[k].dtype, device=dev)
                big[:, off:off + N] = i[k]
                i[k] = big[:, off:off + N]
            w = torch.full((N + off,), float("nan"), dtype=i["weight"].dtype, device=dev)
            w[off:] = i["weight"]
            i["weight"] = w[off:]
            check_norm(i, dtype)


def test_rms_norm_views_shapes_and_empty_rows(dev):
    s = seq()
    i = norm_inputs(dev, torch.bfloat16, torch.bfloat16, 24, 72, 4)
    y, total, rstd = s.rms_norm(i["x"], i["weight"], i["residual"], save=True)
    dx, dw = s.rms_norm_backward(i["dy"], total, rstd, i["weight"], i["ds"])
    for off, pad in ((0, 8), (1, 3), (8, 0)):
        def view(t):
            big = torch.full((24, off + 72 + pad), float("nan"), dtype=t.dtype, device=dev)
            big[:, off:off + 72] = t
            return big[:, off:off + 72]
        v = {k: view(i[k]) for k in ("x", "residual", "dy", "ds")}
        y2, total2, rstd2 = s.rms_norm(v["x"], i["weight"], v["residual"], save=True)
        assert torch.equal(total, total2)
        within(rstd2, rstd, 2 * NORM_Y * rstd.double().cpu(), "rstd")
        within(y2, y, 2 * (NORM_Y + HALF[torch.bfloat16]) * y.double().abs().cpu(), "y")
        dx2, dw2 = s.rms_norm_backward(v["dy"], view(total), rstd, i["weight"], v["ds"])
        within(dx2, dx, 2 * HALF[torch.bfloat16] * dx.double().abs().cpu() + 1e-4, "dx")
        within(dw2, dw, 2 * (52 * U) * 24 * 20 * torch.ones(72), "dw")
    shaped = s.rms_norm(i["x"].view(2, 3, 4, 72), i["weight"], i["residual"].view(2, 3, 4, 72), save=True)
    assert shaped[0].shape == (2, 3, 4, 72) and shaped[2].shape == (2, 3, 4) and torch.equal(shaped[0].view(24, 72), y)
    assert torch.equal(s.rms_norm_backward(i["dy"].view(2, 3, 4, 72), shaped[1], shaped[2], i["weight"], i["ds"].view(2, 3, 4, 72))[1], dw)
    one = s.rms_norm_fp8(i["x"][3], i["weight"], i["residual"][3])
    assert one[0].shape == (72,) and one[1].shape == () and torch.equal(one[2], total[3])
    t = s.rms_norm(i["x"].t().contiguous().t(), i["weight"], i["residual"], save=True)     # channels not contiguous: copied
    assert torch.equal(t[0], y)
    e = i["x"][:0]
    y, total, rstd = s.rms_norm(e, i["weight"], e, save=True)
    dx, dw = s.rms_norm_backward(e, total, rstd, i["weight"])
    assert y.shape == dx.shape == (0, 72) and dw.shape == (72,) and not dw.any()
    assert s.rms_norm_fp8(e, i["weight"])[1].shape == (0,)


def test_rms_norm_more_rows_than_a_launch(dev):
    s = seq()
    R = 2 * 2 ** 21 + 77
    g = torch.Generator(dev).manual_seed(6)
    x, res = (torch.randn(R, 8, generator=g, device=dev).bfloat16() for _ in range(2))
    w = torch.randn(8, generator=g, device=dev).bfloat16()
    y, total, rstd = s.rms_norm(x, w, res, save=True)
    q, scale, _ = s.rms_norm_fp8(x, w, res)
    for a in (0, 2 ** 21 - 50, 2 ** 22 - 50, R - 100):
        c = slice(a, a + 100)
        one = s.rms_norm(x[c], w, res[c], save=True)
        assert torch.equal(y[c], one[0]) and torch.equal(total[c], one[1]) and torch.equal(rstd[c], one[2])
        one = s.rms_norm_fp8(x[c], w, res[c])
        assert torch.equal(q[c].view(torch.uint8), one[0].view(torch.uint8)) and torch.equal(scale[c], one[1])


def test_rms_norm_special_rows(dev):
    """Rows of zeros, of the type's smallest and largest values, with infinities and NaN; each leaves the others alone."""
    s = seq()
    for dtype in DTYPES:
        for N in (64, 72, 2048, 101):
            i = norm_inputs(dev, dtype, None, 7, N, N)
            x, w = i["x"], i["weight"]
            x[1] = 0
            x[2, 5], x[3, 5] = float("nan"), float("inf")
            x[4] = torch.finfo(dtype).smallest_normal
            x[5] = 100.0
            y, _ = s.rms_norm(x, w)
            q, scale, _ = s.rms_norm_fp8(x, w)
            clean = [0, 6]
            y0, _ = s.rms_norm(x[clean], w)
            q0, scale0, _ = s.rms_norm_fp8(x[clean], w)
            assert torch.equal(y[clean], y0) and torch.equal(scale[clean], scale0)
            assert torch.equal(q[clean].view(torch.uint8), q0.view(torch.uint8))
            assert not y[1].any() and float(scale[1]) == 1 and not q[1].float().any()
            assert bool(y[2].isnan().all()) and bool(scale[2].isnan())                 # the whole row's mean is NaN
            assert bool(y[3, 5].isnan()) and not y[3, :5].any() and bool(scale[3].isnan())      # inf / inf, finite / inf
            assert bool(y[4].isfinite().all()) and bool(scale[4].isfinite()) and float(scale[4]) >= 2.0 ** -126
            assert int(q[5].float().abs().max()) == 448
    # a row so small that its scale is at its least value, and y = x / sqrt(eps) = 1000 x: 1000 2^-140 / 2^-126 = 0.06104, and
    # e4m3 has 0.0586 and 0.0625 there
    x = torch.full((1, 64), 2.0 ** -140, device=dev)
    w = torch.ones(64, device=dev)
    q, scale, _ = s.rms_norm_fp8(x, w)
    assert float(scale[0]) == 2.0 ** -126 and bool((q.float() == 0.0625).all())


def test_rms_norm_offsets_beyond_32_bits(dev):
    s = seq()
    R, N, far = 40, 64, 1 << 26
    store = torch.empty((R - 1) * far + N, dtype=torch.bfloat16, device=dev)
    i = norm_inputs(dev, torch.bfloat16, torch.bfloat16, R, N, 3)
    x = torch.as_strided(store, (R, N), (far, 1))
    x.copy_(i["x"])
    for a, b in zip(s.rms_norm(i["x"], i["weight"], i["residual"], save=True), s.rms_norm(x, i["weight"], i["residual"], save=True)):
        assert torch.equal(a, b)
    for a, b in zip(s.rms_norm_backward(i["x"], i["residual"], torch.ones(R, device=dev), i["weight"], i["ds"]),
                    s.rms_norm_backward(x, i["residual"], torch.ones(R, device=dev), i["weight"], i["ds"])):
        assert torch.equal(a, b)


def test_rms_norm_gradient_matches_differences(dev):
    s = seq()
    i = norm_inputs(dev, torch.float32, torch.float32, 40, 100, 8)
    y, total, rstd = s.rms_norm(i["x"], i["weight"], i["residual"], save=True)
    dx, dw = s.rms_norm_backward(i["dy"], total, rstd, i["weight"], i["ds"])
    g = torch.Generator(device=dev).manual_seed(1)
    vx, vw = torch.randn(40, 100, generator=g, device=dev), torch.randn(100, generator=g, device=dev)

    def value(e):
        y, total = s.rms_norm(i["x"] + e * vx, i["weight"] + e * vw, i["residual"])
        return float((y.double() * i["dy"]).sum() + (total.double() * i["ds"]).sum())
    e = 2.0 ** -8
    want, got = float((dx.double() * vx).sum() + (dw.double() * vw).sum()), (value(e) - value(-e)) / (2 * e)
    # 4000 terms of size 4 each off by some 4 U on their own, and the cubic term e^2 of a value of size sqrt(4000) * 3
    assert abs(got - want) <= math.sqrt(4000) * 4 * 8 * U / (2 * e) + math.sqrt(4000) * 3 * e * e, (got, want)


def test_rms_norm_in_graphs(dev):
    s = seq()
    for R, N in ((3, 64), (900, 1000), (70, 4099)):
        i = norm_inputs(dev, torch.bfloat16, torch.float32, R, N, N)

        def train():
            y, total, rstd = s.rms_norm(i["x"], i["weight"], i["residual"], save=True)
            return (y, total) + s.rms_norm_backward(i["dy"], total, rstd, i["weight"], i["ds"])
        replayed(dev, train, list)
        replayed(dev, lambda: s.rms_norm_fp8(i["x"], i["weight"], i["residual"]),
                 lambda o: [o[0].view(torch.uint8), o[1], o[2]])


# -------------------------------------------------------------------------------------------- top-logit distillation
def distill_inputs(dev, dtype, R, V, K, seed, coef=True, absent=0.1, twice=True, tdtype=None, itype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn((R, V), generator=g) * 2.5).to(dtype)
    index = torch.randint(0, V, (R, K), generator=g)
    if twice and K > 2:
        index[:, 1] = index[:, 0]                       # the same column from two slots
    teacher = (torch.randn((R, K), generator=g) * 2 + 4).to(tdtype or dtype)
    gone = torch.rand((R, K), generator=g) < absent
    teacher[gone & (torch.arange(K) % 2 == 0)] = -math.inf
    far = torch.tensor([-1, V, V + 7, 2 ** 31 - 1, -2 ** 31], dtype=torch.int64)[torch.randint(0, 5, (R, K), generator=g)]
    index = torch.where(gone & (torch.arange(K) % 2 == 1), far, index)
    c = torch.rand(R, generator=g) * 2 - 0.5 if coef else None
    if coef and R > 2:
        c[1] = 0
    if R > 3:
        teacher[2] = -math.inf                          # nothing there
        index[3] = -1
    return {k: None if v is None else v.to(dev) for k, v in dict(logits=logits, teacher=teacher, index=index.to(itype), coef=c).items()}


def distill_reference(i, tau):
    x, t, ix = i["logits"].double().cpu() / tau, i["teacher"].double().cpu() / tau, i["index"].cpu().long()
    R, V = x.shape
    ok = (ix >= 0) & (ix < V) & (t > -math.inf)
    c = torch.ones(R, dtype=torch.float64) if i["coef"] is None else i["coef"].double().cpu()
    live = ok.any(1) & (c != 0)
    q = torch.softmax(torch.where(ok, t, torch.tensor(-1e300, dtype=torch.float64)), 1) * ok
    logp = torch.log_softmax(x, 1)
    lp = logp.gather(1, ix.clamp(0, V - 1))
    each = torch.where(q > 0, q * (torch.log(q.clamp_min(1e-320)) - lp), torch.zeros_like(q))
    d = torch.exp(logp).scatter_add(1, ix.clamp(0, V - 1), -q)
    zero = torch.zeros((), dtype=torch.float64)
    loss = torch.where(live, c * tau * tau * each.sum(1), zero)
    return loss, torch.where(live[:, None], (c * tau)[:, None] * d, zero), q, lp, c


def check_distill(i, dtype, tau):
    s = seq()
    loss, d = s.topk_distill(i["logits"], i["teacher"], i["index"], temperature=tau, coef=i["coef"])
    loss2, none = s.topk_distill(i["logits"], i["teacher"], i["index"], temperature=tau, coef=i["coef"], grad=False)
    assert none is None and torch.equal(loss, loss2) and d.dtype == dtype and loss.dtype == torch.float32
    rl, rd, q, lp, c = distill_reference(i, tau)
    V, span = i["logits"].shape[1], float((i["logits"].double().max() - i["logits"].double().min()) / tau)
    # an exponent (x - m) k2 of at most `span` nats has three roundings (the difference, k2, the product); the sum's terms 8
    # columns a step and at most 80 steps a thread, the joins 10 more; exp2, the reciprocal and two products 1 ulp each
    rel = (3 * span + 8 + 90 + 10) * U
    p = (rd / (c * tau)[:, None].where((c != 0)[:, None], torch.ones(1, dtype=torch.float64))).abs()
    qcol = torch.zeros_like(rd).scatter_add(1, i["index"].cpu().long().clamp(0, V - 1), q)
    tol = (c.abs() * tau)[:, None] * (rel * (p + 2 * qcol) + 1e-37) + HALF[dtype] * rd.abs() + (SMALL if dtype == torch.float16 else 2.0 ** -134)
    within(d, rd, tol, "dlogits")
    tspan = float(i["teacher"].double().abs().nan_to_num(posinf=0).max()) / tau
    # log q and log p of a size up to span + log V, each with the roundings above, weights q with those of K <= 512 slots
    size = span + tspan + math.log(V) + 7
    within(loss, rl, c.abs() * tau * tau * (rel + (3 * tspan + 30) * U + 6 * U) * size * (q.sum(1) + 1e-30), "loss")
    inplace = i["logits"].clone()
    loss3, d3 = s.topk_distill(inplace, i["teacher"], i["index"], temperature=tau, coef=i["coef"], out=inplace)
    assert d3 is inplace and torch.equal(loss3, loss) and torch.equal(d3, d)


DISTILL_SIZES = [(1, 1, 1), (5, 3, 2), (4, 17, 5), (6, 64, 64), (300, 256, 8), (3, 257, 9), (7, 1000, 33), (2, 2048, 512), (5, 4099, 100),
                 (2, 8192, 16), (130, 8200, 16), (2, 16387, 100), (131, 20001, 20), (2, 32768, 3), (129, 40003, 50), (1, 65536, 64), (3, 131072, 128),
                 (130, 131075, 40), (2, 163840, 30), (129, 163841, 7), (2, 200003, 77),
                 (20000, 101, 20), (16000, 520, 64), (15000, 9, 3), (8000, 1500, 65)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("R,V,K", DISTILL_SIZES)
def test_topk_distill_matches_its_formulas(dev, dtype, R, V, K):
    tau = (1.0, 0.5, 2.0, 3.7)[(R + V + K) % 4]
    check_distill(distill_inputs(dev, dtype, R, V, K, V + K, tdtype=(None, torch.float32)[V % 2],
                                 itype=(torch.int64, torch.int32)[K % 2], coef=V % 3 > 0), dtype, tau)


def test_topk_distill_views_and_misaligned_rows(dev):
    """Row strides and offsets of every distance to a 16-byte boundary, in and out at different ones, expanded teachers."""
    s = seq()
    for dtype in (torch.float32, torch.bfloat16):
        for V in (40, 1001, 3000, 70001):
            i = distill_inputs(dev, dtype, 6, V, 12, V)
            want = s.topk_distill(i["logits"], i["teacher"], i["index"], 1.5, i["coef"])
            rl, rd, q, lp, c = distill_reference(i, 1.5)
            for off, pad, ooff, opad in ((1, 0, 1, 0), (3, 5, 3, 5), (0, 1, 2, 3), (7, 8, 0, 0)):
                big = torch.full((6, off + V + pad), float("nan"), dtype=dtype, device=dev)
                x = big[:, off:off + V]
                x.copy_(i["logits"])
                buf = torch.full((6, ooff + V + opad), 7.0, dtype=dtype, device=dev)
                out = buf[:, ooff:ooff + V]
                loss, d = s.topk_distill(x, i["teacher"], i["index"], 1.5, i["coef"], out=out)
                # twice the tolerance of one result: both are within it of the formulas'
                within(loss, want[0], 1e-4 * (1 + want[0].double().abs().cpu()), "loss")
                within(d, want[1], 2e-5 + 2 * HALF[dtype] * want[1].double().abs().cpu(), "dlogits")
                assert bool((buf[:, :ooff] == 7).all()) and bool((buf[:, ooff + V:] == 7).all())
                assert bool(x.isfinite().all())
    i = distill_inputs(dev, torch.float32, 5, 300, 6, 1, absent=0)
    one = s.topk_distill(i["logits"][:1], i["teacher"][:1], i["index"][:1])
    more = s.topk_distill(i["logits"][:1].expand(5, 300), i["teacher"][:1].expand(5, 6), i["index"][:1].expand(5, 6))
    assert torch.equal(more[0], one[0].expand(5)) and torch.equal(more[1], one[1].expand(5, 300))
    t = s.topk_distill(i["logits"].t().contiguous().t(), i["teacher"], i["index"])
    assert torch.equal(t[1], s.topk_distill(i["logits"], i["teacher"], i["index"])[1])


@pytest.mark.parametrize("R,V", [(8, 64), (8, 1500), (8, 9001), (200, 9001), (8, 70000), (200, 70000), (8, 170000)])
def test_topk_distill_masks_infinities_and_nan(dev, R, V):
    s = seq()
    for dtype in DTYPES:
        i = distill_inputs(dev, dtype, R, V, 6, V, coef=False, absent=0, twice=False)
        x, t, ix = i["logits"], i["teacher"], i["index"]
        t[2] = 1.0
        for r in range(R):
            ix[r] = torch.tensor([0, 3, 5, 9, V - 1, V // 2], device=dev)
        base = s.topk_distill(x, t, ix)
        coef = torch.ones(R, device=dev)
        coef[0], t[1], ix[4] = 0, -math.inf, V                   # three ways to be left out
        x[0], x[1] = float("nan"), float("inf")
        x[4] = -math.inf
        low = torch.finfo(dtype).min
        x[3, :] = low                                            # nothing but the mask: uniform
        x[5, 20:] = low                                          # masked columns, some the teacher's
        x[6, 20:] = -math.inf
        t[6, 4:] = -math.inf
        x[7, 11] = float("nan")
        loss, d = s.topk_distill(x, t, ix, coef=coef)
        for r in (0, 1, 4):
            assert float(loss[r]) == 0 and not d[r].any()
        for r in [2] + list(range(8, R)):
            assert torch.equal(loss[r], base[0][r]) and torch.equal(d[r], base[1][r])
        cols = torch.ones(V, dtype=torch.bool, device=dev)
        cols[ix[3]] = False
        within(d[3][cols], torch.full((int(cols.sum()),), 1 / V), (HALF[dtype] + 200 * U) / V + SMALL, "uniform")
        assert not d[5, 20:V // 2].any() and not d[6, 20:].any()
        # the teacher's two masked columns cost q |low| each (log p = low - log of the sum), the others a few nats
        masked = float(torch.softmax(t[5].double(), 0)[4:].sum())
        assert float(loss[5]) >= 0.99 * masked * -low - 100 and bool(loss[6].isfinite()) and bool(d[5].isfinite().all())
        assert bool(loss[7].isnan()) and bool(d[7].isnan().all())
        xi = x.clone()
        loss2, d2 = s.topk_distill(xi, t, ix, coef=coef, out=xi)
        assert torch.equal(loss2.nan_to_num(5), loss.nan_to_num(5)) and torch.equal(d2.nan_to_num(5), d.nan_to_num(5))
        # a student that rules the teacher's column out: the loss is infinite, the gradient -q there
        x[2, 9] = -math.inf
        loss, d = s.topk_distill(x[2:3], t[2:3], ix[2:3])
        assert float(loss) == math.inf and abs(float(d[0, 9]) + 1 / 6) <= HALF[dtype] / 6 + 1e-6
        t[2, 0] = float("nan")
        loss, d = s.topk_distill(x[2:3], t[2:3], ix[2:3])
        assert bool(loss.isnan().all()) and bool(d[0, ix[2]].isnan().all())


def test_topk_distill_gradient_matches_differences(dev):
    s = seq()
    for V in (50, 3000, 40000):
        i = distill_inputs(dev, torch.float32, 8, V, 16, V)
        loss, d = s.topk_distill(i["logits"], i["teacher"], i["index"], 2.0, i["coef"])
        v = torch.randn(8, V, generator=torch.Generator(device=dev).manual_seed(1), device=dev)

        def value(e):
            return float(s.topk_distill(i["logits"] + e * v, i["teacher"], i["index"], 2.0, i["coef"], grad=False)[0].double().sum())
        e = 2.0 ** -6
        want, got = float((d.double() * v).sum()), (value(e) - value(-e)) / (2 * e)
        # 8 rows of losses up to 2 * 4 * 20, off by some 100 U each, and the cubic term of tau^2 log-sum-exp: e^2 |v|^3 / tau
        assert abs(got - want) <= 8 * 160 * 100 * U / (2 * e) + 8 * 2 * e * e * 8, (V, got, want)


def test_topk_distill_no_rows_and_offsets_beyond_32_bits(dev):
    s = seq()
    e = torch.empty((0, 50), device=dev)
    loss, d = s.topk_distill(e, e[:, :4], e[:, :4].long())
    assert loss.shape == (0,) and d.shape == (0, 50)
    far = 1 << 26
    for V in (100, 12000):
        i = distill_inputs(dev, torch.bfloat16, 40, V, 6, 2)
        store = torch.empty(39 * far + V, dtype=torch.bfloat16, device=dev)
        x = torch.as_strided(store, (40, V), (far, 1))
        x.copy_(i["logits"])
        want = s.topk_distill(i["logits"], i["teacher"], i["index"], 1.0, i["coef"])
        loss, d = s.topk_distill(x, i["teacher"], i["index"], 1.0, i["coef"])
        # rows at another distance to a 16-byte boundary are summed in another order: each result is within half a step of the
        # formulas' and what 32 bits lose (as in check_distill, below 2^-15 of p <= 1 and of the loss for these spans)
        for again in range(2):
            within(loss, want[0], 2.0 ** -14 * (1 + want[0].double().abs().cpu()), "loss")
            within(d, want[1], 2.0 ** -14 + 2 * HALF[torch.bfloat16] * want[1].double().abs().cpu(), "dlogits")
            if not again:
                loss, d = s.topk_distill(x, i["teacher"], i["index"], 1.0, i["coef"], out=x)
                assert d is x


def test_topk_distill_in_graphs(dev):
    s = seq()
    for R, V in ((64, 256), (3, 50000), (300, 5001), (3, 140001)):
        i = distill_inputs(dev, torch.bfloat16, R, V, 10, V)
        replayed(dev, lambda: s.topk_distill(i["logits"], i["teacher"], i["index"], 1.0, i["coef"]), list)


# ------------------------------------------------------------------------------------------------ all of them
def test_rows_of_any_stride(dev):
    """Broadcast steps (stride 0), windows that overlap (a stride below the width), single channels of wider rows."""
    s = seq()
    for dtype in (torch.float32, torch.bfloat16):
        for T in (3, 40, 300):
            for D in (1, 16, 50):
                i = scan_inputs(dev, dtype, 2, T, D, T + D)
                base = torch.randn((2, T + D), device=dev).to(dtype)
                windows = torch.as_strided(base, (2, T, D), (T + D, 1, 1))
                fixed = i["gate"][:, :1].expand(2, T, D)
                one = torch.randn((2, T, D, 3), device=dev).to(dtype)[..., 1]
                for gate, x in ((fixed, windows), (i["gate"], windows), (windows, i["x"]), (one, one)):
                    a = s.gated_scan(gate, x, i["h0"], save=True)
                    b = s.gated_scan(gate.contiguous(), x.contiguous(), i["h0"], save=True)
                    ga = s.gated_scan_backward(gate, x, a[2], i["dy"], i["dh_last"])
                    gb = s.gated_scan_backward(gate.contiguous(), x.contiguous(), b[2], i["dy"], i["dh_last"])
                    # narrow and wide loads join in another order: both within check_scan's tolerance, |G| <= 57 * 5, |h| + |x| <= 10
                    for u, v in zip(a + ga, b + gb):
                        within(u, v, 2 * (2 * SCAN_STATE * 57 * 5 * 10 / 4 + HALF[dtype] * v.double().abs().cpu()), "strides")
    x = torch.randn((1, 96), device=dev).bfloat16().expand(5, 96)
    w = torch.ones(96, device=dev)
    y, total, rstd = s.rms_norm(x, w, residual=x, save=True)
    assert torch.equal(y, y[:1].expand(5, 96)) and torch.equal(total, (x.float() * 2).bfloat16())
    dx, dw = s.rms_norm_backward(x, total, rstd, w, ds=x)
    assert torch.equal(dx, dx[:1].expand(5, 96))


def test_one_step_whose_time_stride_means_nothing(dev):
    """(B, 1, D) tensors made by a transpose have a time stride of one element."""
    s = seq()
    g = torch.Generator(dev).manual_seed(2)
    for dtype, D in ((torch.float32, 48), (torch.bfloat16, 130), (torch.bfloat16, 3)):
        gate, x, dy = (torch.randn(5, 1, D, generator=g, device=dev).to(dtype) for _ in range(3))
        y, h, saved = s.gated_scan(gate, x, save=True)
        want = s.gated_scan_backward(gate, x, saved, dy)
        flat = lambda t: t.reshape(5, D).clone().view(5, D, 1).transpose(1, 2)
        assert flat(x).stride() == (D, 1, 1)
        y2, h2, saved2 = s.gated_scan(flat(gate), flat(x), save=True)
        assert torch.equal(y, y2) and torch.equal(h, h2) and torch.equal(saved, saved2)
        out = tuple(torch.full((5, D, 1), 9.0, dtype=dtype, device=dev).transpose(1, 2) for _ in range(2))
        got = s.gated_scan_backward(flat(gate), flat(x), saved, flat(dy), out=out)
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dtype,B,T,D", [(torch.bfloat16, 64, 1024, 1024), (torch.bfloat16, 4, 8192, 2048), (torch.float32, 12, 1024, 4096),
                                         (torch.float16, 8192, 16, 1024)], ids=str)
def test_gated_scan_larger_than_the_caches(dev, dtype, B, T, D):
    """The same bits as with rows that lie otherwise in memory, which are not streamed past the caches."""
    s = seq()
    g = torch.Generator(dev).manual_seed(B)
    r = lambda: torch.randn(B, T, D, generator=g, device=dev, dtype=torch.float32).to(dtype)
    gate, x, dy = r(), r(), r()
    starts = torch.rand(B, T, generator=g, device=dev) < 0.01
    lengths = torch.randint(0, T + 1, (B,), generator=g, device=dev)

    def other(t):
        big = torch.empty(B, T, D + 4, dtype=dtype, device=dev)
        big[:, :, :D] = t
        return big[:, :, :D]
    y, h = s.gated_scan(gate, x, starts=starts, lengths=lengths)
    y2, h2, saved = s.gated_scan(gate, x, starts=starts, lengths=lengths, save=True)
    y3, h3, saved3 = s.gated_scan(other(gate), x, starts=starts, lengths=lengths, save=True)
    assert torch.equal(y, y3) and torch.equal(y2, y3) and torch.equal(h, h3) and torch.equal(h2, h3) and torch.equal(saved, saved3)
    one = s.gated_scan_backward(gate, x, saved, dy, starts=starts, lengths=lengths)
    two = s.gated_scan_backward(gate, other(x), saved, dy, starts=starts, lengths=lengths)
    assert all(torch.equal(p, q) for p, q in zip(one, two))


@pytest.mark.parametrize("dtype,R,N", [(torch.bfloat16, 12288, 4096), (torch.float32, 12000, 4096), (torch.float16, 700000, 128)], ids=str)
def test_rms_norm_larger_than_the_caches(dev, dtype, R, N):
    """The same bits as the calls on some of the rows, which are not streamed past the caches."""
    s = seq()
    g = torch.Generator(dev).manual_seed(R)
    r = lambda *n: torch.randn(*n, generator=g, device=dev).to(dtype)
    x, res, dy, ds, w = r(R, N), r(R, N), r(R, N), r(R, N), r(N)
    y, total, rstd = s.rms_norm(x, w, res, save=True)
    q, scale, total2 = s.rms_norm_fp8(x, w, res)
    dx, dw = s.rms_norm_backward(dy, total, rstd, w, ds)
    assert torch.equal(total, total2)
    step, sums = R // 10, []
    for a in range(0, R, step):
        c = slice(a, a + step)
        y1, t1, r1 = s.rms_norm(x[c], w, res[c], save=True)
        q1, s1, _ = s.rms_norm_fp8(x[c], w, res[c])
        d1, w1 = s.rms_norm_backward(dy[c], t1, r1, w, ds[c])
        sums.append(w1.double())
        assert torch.equal(y[c], y1) and torch.equal(total[c], t1) and torch.equal(rstd[c], r1) and torch.equal(dx[c], d1)
        assert torch.equal(q[c].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(scale[c], s1)
    # |dy xh| of a column sums to less than R at unit variance; both sums as in check_norm, of the same terms
    within(dw, sum(sums).cpu(), 2 * (R / 128 + 52) * U * R * torch.ones(N, dtype=torch.float64), "dweight")


def test_topk_distill_larger_than_the_caches(dev):
    s = seq()
    for dtype, R, V in ((torch.bfloat16, 1400, 65536), (torch.float32, 12000, 4096)):
        i = distill_inputs(dev, dtype, R, V, 20, 3)
        loss, d = s.topk_distill(i["logits"], i["teacher"], i["index"], 1.5, i["coef"])
        for a in range(0, R, R // 5):
            c = slice(a, a + R // 5)
            l1, d1 = s.topk_distill(i["logits"][c], i["teacher"][c], i["index"][c], 1.5, i["coef"][c])
            assert torch.equal(loss[c], l1) and torch.equal(d[c], d1)


def test_two_streams_at_once(dev):
    """The same calls on two streams together, those with scratch memory among them, give what one call alone gives."""
    s = seq()
    i = scan_inputs(dev, torch.bfloat16, 2, 3000, 64, 1, starts=True)
    n = norm_inputs(dev, torch.bfloat16, torch.bfloat16, 900, 520, 1)
    k = distill_inputs(dev, torch.bfloat16, 4, 140000, 20, 1)

    def work():
        y, h, saved = s.gated_scan(i["gate"], i["x"], i["h0"], i["starts"], save=True)
        out = [y, h, *s.gated_scan_backward(i["gate"], i["x"], saved, i["dy"], i["dh_last"], i["starts"])]
        y, total, rstd = s.rms_norm(n["x"], n["weight"], n["residual"], save=True)
        out += [y, *s.rms_norm_backward(n["dy"], total, rstd, n["weight"], n["ds"])]
        return out + list(s.topk_distill(k["logits"], k["teacher"], k["index"], 1.0, k["coef"]))
    want = work()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(dev) for _ in range(2)], []
    for _ in range(6):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(work())
    torch.cuda.synchronize()
    for out in got:
        for u, v in zip(out, want):
            assert torch.equal(u, v)


# --------------------------------------------------------------------------------------------------- used together
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_a_recurrent_policy_learns_a_step_from_its_teacher(dev, dtype):
    """norm -> projection -> recurrence -> norm of the residual stream -> logits -> distillation loss, and all the way back,
    against the same network by autograd in 64 bits; and the trained direction lowers the loss."""
    s = seq()
    B, T, D, V, K = 3, 70, 32, 40, 5
    g = torch.Generator().manual_seed(0)
    r = lambda *sh, sc=1.0: (torch.randn(sh, generator=g) * sc).to(dtype).to(dev)  # noqa: E731
    x, w1, w2 = r(B, T, D), 1 + r(D, sc=0.2), 1 + r(D, sc=0.2)
    proj, head = r(D, 2 * D, sc=D ** -0.5), r(D, V, sc=D ** -0.5)
    teacher, index = r(B * T, K, sc=2.0), torch.randint(0, V, (B * T, K), generator=g).to(dev)
    starts = (torch.rand((B, T), generator=g) < 0.1).to(dev)
    coef = torch.full((B * T,), 1.0 / (B * T), device=dev)

    def forward(x):
        n1, s1, r1 = s.rms_norm(x, w1, save=True)
        both = n1 @ proj
        gate, cand = both[..., :D], both[..., D:]
        y, h, saved = s.gated_scan(gate, cand, starts=starts, save=True)
        n2, s2, r2 = s.rms_norm(y, w2, residual=x, save=True)
        logits = (n2 @ head).view(B * T, V)
        return locals()
    f = forward(x)
    loss, dlogits = s.topk_distill(f["logits"], teacher, index, 1.5, coef)
    dn2 = (dlogits @ head.t()).view(B, T, D)
    ds2, dw2 = s.rms_norm_backward(dn2, f["s2"], f["r2"], w2)
    dboth = torch.empty_like(f["both"])
    s.gated_scan_backward(f["gate"], f["cand"], f["saved"], ds2, starts=starts, out=(dboth[..., :D], dboth[..., D:]))
    dx, dw1 = s.rms_norm_backward(dboth @ proj.t(), f["s1"], f["r1"], w1, ds=ds2)

    X, W1, W2, P, H = (t.double().cpu().requires_grad_() for t in (x, w1, w2, proj, head))
    n1 = X / torch.sqrt((X * X).mean(-1, keepdim=True) + 1e-6) * W1
    both = n1 @ P
    h, ys = torch.zeros((B, D), dtype=torch.float64), []
    for t in range(T):
        h = torch.where(starts[:, t, None].cpu(), torch.zeros_like(h), h)
        fg = torch.sigmoid(both[:, t, :D])
        h = fg * h + (1 - fg) * both[:, t, D:]
        ys.append(h)
    s2 = X + torch.stack(ys, 1)
    logits = ((s2 / torch.sqrt((s2 * s2).mean(-1, keepdim=True) + 1e-6) * W2) @ H).view(B * T, V)
    q = torch.softmax(teacher.double().cpu() / 1.5, 1)
    lp = torch.log_softmax(logits / 1.5, 1).gather(1, index.cpu())
    total = (1.5 ** 2 * (q * (torch.log(q) - lp)).sum(1)).mean()
    gx, gw1, gw2 = torch.autograd.grad(total, (X, W1, W2))
    # seven stored tensors each way, a relative error of half a step each, and fp32's sums: 40 half steps of the largest gradient
    tol = 40 * max(HALF[dtype], 16 * U)
    for got, want in ((dx, gx), (dw1, gw1), (dw2, gw2)):
        within(got, want, tol * want.abs().max(), "gradient")
    assert abs(float(loss.sum()) - total.item()) <= tol * total.item()
