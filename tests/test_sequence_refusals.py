"""Calls of the operators of sequence policies that could only give wrong results are refused before anything is launched (no GPU
needed: the pointers are never followed)."""
import pytest

from serl_amd import ops


def norm_fwd(**k):
    return ops.rms_norm_fwd(*{**dict(dtype=1, stream=1, weight=1, R=4, N=8, x=16, ldx=8, residual=32, ldres=8, w=48, eps=1e-6, y=64, ldy=8,
                                     y_fp8=0, scale=None, sum=80, ldsum=8, rstd=None, st=0), **k}.values())


def norm_bwd(**k):
    return ops.rms_norm_bwd(*{**dict(dtype=1, stream=1, weight=1, R=4, N=8, dy=16, lddy=8, sum=32, ldsum=8, rstd=48, w=64, ds=80, ldds=8,
                                     dx=96, lddx=8, dw=112, ws=None, n=0, st=0), **k}.values())


def test_norm_in_place_at_another_row_stride():
    for kw in (dict(y=16, ldy=9), dict(y=16, ldx=16), dict(y=16, ldx=0), dict(sum=32, ldsum=12), dict(sum=32, ldres=0),
               dict(y=16, y_fp8=1, scale=96), dict(y=16, y_fp8=1, scale=96, ldy=8, ldx=8), dict(y=16, y_fp8=1, scale=96, ldy=16, ldx=16)):
        with pytest.raises(ValueError, match="in place needs the same row stride"):
            norm_fwd(**kw)
    for kw in (dict(dx=80, lddx=9), dict(dx=80, ldds=0), dict(dx=32, ldsum=16), dict(dx=32, ds=None, ldsum=0)):
        with pytest.raises(ValueError, match="in place needs the same row stride"):
            norm_bwd(**kw)
    # rows at the same addresses go on to the next check, the workspace's
    for kw in (dict(dx=80), dict(dx=32), dict(dx=32, ldsum=9, lddx=9), dict(R=1, dx=80, lddx=9)):
        with pytest.raises(ValueError, match="workspace"):
            norm_bwd(**kw)


def distill(**k):
    return ops.topk_distill(*{**dict(dtype=1, tt=1, i64=1, R=4, V=9, K=3, logits=16, ldl=0, teacher=16, ldt=0, index=16, ldi=0, tau=1.0,
                                     coef=None, loss=16, d=None, ldd=0, ws=16, n=1 << 60, st=0), **k}.values())


def test_distillation_of_more_long_rows_than_a_launch():
    """Expanded logits alone make so many: rows of 163 841 16-bit columns are cut in 6 pieces of 320 threads."""
    most = (2 ** 32 - 1) // 320 // 6
    for R in (most + 1, 2 ** 24, 2 ** 31 - 2 ** 16):
        with pytest.raises(ValueError, match=f"too many rows of this length: R at most {most}"):
            distill(R=R, V=163841)
    with pytest.raises(ValueError, match="R at most"):
        distill(dtype=0, tt=0, R=2 ** 24, V=2 ** 29)


def scan_fwd(**k):
    return ops.gated_scan_fwd(*{**dict(dtype=0, B=2, T=5000, D=8, gate=16, gate_bs=40000, gate_ts=8, x=16, x_bs=40000, x_ts=8, h0=None, starts=None,
                                       starts_bs=0, lengths=None, y=16, y_bs=40000, y_ts=8, h_last=16, states=None, ws=None, n=0, st=0), **k}.values())


def scan_bwd(**k):
    return ops.gated_scan_bwd(*{**dict(dtype=0, B=2, T=5000, D=8, gate=16, gate_bs=40000, gate_ts=8, x=16, x_bs=40000, x_ts=8, starts=None,
                                       starts_bs=0, lengths=None, states=16, dy=16, dy_bs=40000, dy_ts=8, dh_last=None, dgate=1 << 20,
                                       dgate_bs=40000, dgate_ts=8, dx=1 << 21, dx_bs=40000, dx_ts=8, dh0=16, ws=None, n=0, st=0), **k}.values())


def test_recurrence_whose_outputs_share_memory():
    # rows of one output: sequences a step apart, the last step over the next sequence's first
    for bs, ts in ((8, 8), (39996, 8), (7, 40000), (8, 15), (0, 8), (40000, 0)):
        with pytest.raises(ValueError, match="rows of y overlap"):
            scan_fwd(y_bs=bs, y_ts=ts)
        with pytest.raises(ValueError, match="rows of dgate or dx overlap"):
            scan_bwd(dgate_bs=bs, dgate_ts=ts)
        with pytest.raises(ValueError, match="rows of dgate or dx overlap"):
            scan_bwd(dx_bs=bs, dx_ts=ts)
    # the two outputs over each other: the same tensor, halves that are not apart, one a step or a sequence on, time-major ones
    at, half = 1 << 20, dict(dgate_bs=80000, dgate_ts=16, dx_bs=80000, dx_ts=16)
    for kw in (dict(dx=at), dict(dx=at, dx_ts=16, dx_bs=80000), dict(dx=at + 4), dict(dx=at + 32 * 4999), dict(dx=at - 32), dict(dx=at + 40000 * 4),
               dict(half, dx=at + 28), dict(half, dx=at + 64 * 17 - 4), dict(half, dx=at - 80000 * 4 + 64),
               dict(dgate_bs=8, dgate_ts=16, dx_bs=8, dx_ts=16, dx=at + 32)):
        with pytest.raises(ValueError, match="rows of dgate or dx overlap"):
            scan_bwd(**kw)
    # outputs that lie apart go on to the next check, the workspace's
    for kw in (dict(), dict(half, dx=at + 32), dict(half, dx=at - 32), dict(half, dx=at + 64 * 17 + 32), dict(dx=at + 40000 * 2 * 4),
               dict(dgate_bs=8, dgate_ts=32, dx_bs=8, dx_ts=32, dx=at + 64)):
        with pytest.raises(ValueError, match="workspace"):
            scan_bwd(**kw)
    for bs, ts in ((40000, 8), (8, 16), (8, 64), (80000, 16)):
        with pytest.raises(ValueError, match="workspace"):
            scan_fwd(y_bs=bs, y_ts=ts)
    with pytest.raises(ValueError, match="h_last may be h0 for up to 8 steps"):
        scan_fwd(h0=16)
