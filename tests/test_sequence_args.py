"""What the operators of sequence policies refuse, and how: checked before anything reaches a device (no GPU needed)."""
import pytest
import torch

from serl_amd import ops, sequence


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def test_gated_scan_refusals():
    g = t(2, 5, 8)
    with pytest.raises(ValueError, match=r"gate must be a \(B, T, D\)"):
        sequence.gated_scan(t(2, 8), t(2, 8))
    with pytest.raises(ValueError, match="x must have the shape"):
        sequence.gated_scan(g, t(2, 5, 7))
    with pytest.raises(TypeError, match="gate must be float32"):
        sequence.gated_scan(g.double(), g.double())
    with pytest.raises(TypeError, match="x must be"):
        sequence.gated_scan(g, g.half())
    with pytest.raises(TypeError, match="x must be a tensor"):
        sequence.gated_scan(g, None)
    with pytest.raises(ValueError, match="h0 must have the shape"):
        sequence.gated_scan(g, g, h0=t(2, 9))
    with pytest.raises(TypeError, match="h0 must be"):
        sequence.gated_scan(g, g, h0=t(2, 8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="starts must have the shape"):
        sequence.gated_scan(g, g, starts=t(2, 4, dtype=torch.bool))
    with pytest.raises(TypeError, match="starts must be"):
        sequence.gated_scan(g, g, starts=t(2, 5))
    with pytest.raises(TypeError, match="lengths must be"):
        sequence.gated_scan(g, g, lengths=t(2))
    with pytest.raises(TypeError, match="gate must be a CUDA tensor"):
        sequence.gated_scan(g, g)
    with pytest.raises(ValueError, match="saved must have the shape"):
        sequence.gated_scan_backward(g, g, t(2, 2, 8), g)
    with pytest.raises(ValueError, match="dy must have the shape"):
        sequence.gated_scan_backward(g, g, t(2, 1, 8), t(2, 5, 9))
    with pytest.raises(TypeError, match=r"out\[0\] must be"):
        sequence.gated_scan_backward(g, g, t(2, 1, 8), g, out=(g.half(), g))
    with pytest.raises(ValueError, match="contiguous channels"):
        sequence.gated_scan_backward(g, g, t(2, 1, 8), g, out=(t(2, 8, 5).transpose(1, 2), g))
    with pytest.raises(ValueError, match=r"gate must be a \(B, D\)"):
        sequence.gated_scan_step(g, g, t(2, 8))
    with pytest.raises(TypeError, match="h must be a tensor"):
        sequence.gated_scan_step(t(2, 8), t(2, 8), None)
    with pytest.raises(ValueError, match="h_out must be contiguous"):
        sequence.gated_scan_step(t(2, 8), t(2, 8), t(2, 8), h_out=t(8, 2).t())


def test_gated_scan_entry_point_refusals():
    scan = lambda **k: ops.gated_scan_fwd(*{**dict(  # noqa: E731
        dtype=0, B=2, T=5, D=8, gate=16, gate_bs=40, gate_ts=8, x=16, x_bs=40, x_ts=8, h0=None, starts=None, starts_bs=0,
        lengths=None, y=16, y_bs=40, y_ts=8, h_last=16, states=None, workspace=None, workspace_bytes=0, stream=0), **k}.values())
    with pytest.raises(ValueError, match="type must be"):
        scan(dtype=3)
    with pytest.raises(ValueError, match="negative size"):
        scan(T=-1)
    with pytest.raises(ValueError, match="null pointer"):
        scan(x=None)
    with pytest.raises(ValueError, match="negative stride"):
        scan(gate_ts=-8)
    with pytest.raises(ValueError, match="rows of y overlap"):
        scan(y_ts=4)
    with pytest.raises(ValueError, match="D must be at most 67108864"):
        scan(D=(1 << 26) + 1)
    with pytest.raises(ValueError, match="15 steps of a tensor must span less than"):
        scan(T=9, gate_ts=1 << 26)
    with pytest.raises(ValueError, match=r"workspace of \d+ bytes needed, 0 available"):
        scan(T=5000, gate_bs=40000, x_bs=40000, y_bs=40000)
    for many in (dict(B=1 << 27, T=16), dict(B=1 << 24, T=60), dict(B=1 << 29, T=1, D=64, y_ts=64, y_bs=64),
                 dict(B=1 << 23, T=100, D=2)):                    # a launch of 2^32 threads or more
        with pytest.raises(ValueError, match=r"B \* D too large"):
            scan(**many)
    with pytest.raises(ValueError, match="bad type or sizes"):
        ops.gated_scan_workspace_bytes(9, 1, 1, 1)
    with pytest.raises(ValueError, match="bad sizes"):
        ops.gated_scan_states_floats(1, -1, 1)
    assert ops.gated_scan_workspace_bytes(1, 8, 4096, 2048) == 0
    assert ops.gated_scan_states_floats(2, 129, 8) == 2 * 3 * 8
    bwd = lambda **k: ops.gated_scan_bwd(*{**dict(  # noqa: E731
        dtype=0, B=2, T=5, D=8, gate=16, gate_bs=40, gate_ts=8, x=16, x_bs=40, x_ts=8, starts=None, starts_bs=0, lengths=None,
        states=16, dy=16, dy_bs=40, dy_ts=8, dh_last=None, dgate=16, dgate_bs=40, dgate_ts=8, dx=16, dx_bs=40, dx_ts=8, dh0=16,
        workspace=None, workspace_bytes=0, stream=0), **k}.values())
    with pytest.raises(ValueError, match="T must be >= 1"):
        bwd(T=0)
    with pytest.raises(ValueError, match="null pointer"):
        bwd(states=None)
    with pytest.raises(ValueError, match="rows of dgate or dx overlap"):
        bwd(dx_bs=4)
    with pytest.raises(ValueError, match=r"B \* D too large"):
        bwd(B=1 << 26)


def test_rms_norm_refusals():
    x, w = t(4, 8), t(8)
    with pytest.raises(ValueError, match=r"x must be a \(\.\.\., N\) tensor"):
        sequence.rms_norm(t(), w)
    with pytest.raises(ValueError, match="N must be in"):
        sequence.rms_norm(t(4, 0), t(0))
    with pytest.raises(ValueError, match="N must be in"):
        sequence.rms_norm_fp8(t(1, 32769), t(32769))
    with pytest.raises(TypeError, match="x must be float32"):
        sequence.rms_norm(x.double(), w)
    with pytest.raises(ValueError, match="weight must have the shape"):
        sequence.rms_norm(x, t(9))
    with pytest.raises(TypeError, match="weight must be"):
        sequence.rms_norm(x.half(), w.bfloat16())
    with pytest.raises(ValueError, match="residual must have the shape"):
        sequence.rms_norm(x, w, residual=t(3, 8))
    with pytest.raises(TypeError, match="residual must be"):
        sequence.rms_norm(x, w, residual=x.half())
    with pytest.raises(TypeError, match="x must be a CUDA tensor"):
        sequence.rms_norm(x, w)
    with pytest.raises(ValueError, match="rstd must have the shape"):
        sequence.rms_norm_backward(x, x, t(5), w)
    with pytest.raises(TypeError, match="ds must be"):
        sequence.rms_norm_backward(x.half(), x, t(4), w, ds=x.half())
    with pytest.raises(TypeError, match="s must be"):
        sequence.rms_norm_backward(x, x.half(), t(4), w)
    fwd = lambda **k: ops.rms_norm_fwd(*{**dict(  # noqa: E731
        dtype=1, stream=1, weight=1, R=4, N=8, x=16, ldx=8, residual=16, ldres=8, w=16, eps=1e-6, y=16, ldy=8, y_fp8=0,
        scale=None, sum=16, ldsum=8, rstd=None, st=0), **k}.values())
    for match, kw in (("type must be", dict(dtype=5)), ("residual's type", dict(stream=2)), ("weight's type", dict(weight=2)),
                      ("N must be", dict(N=0)), ("N must be", dict(R=-1)), ("null pointer", dict(w=None)),
                      ("go together", dict(sum=None)), ("its type is x's", dict(residual=None, sum=None, stream=0)),
                      ("scales' buffer", dict(y_fp8=1)), ("overlap", dict(ldy=7)), ("negative", dict(ldx=-8))):
        with pytest.raises(ValueError, match=match):
            fwd(**kw)
    with pytest.raises(ValueError, match=r"workspace of 128 bytes needed, 127 available"):
        ops.rms_norm_bwd(1, 1, 1, 4, 8, 16, 8, 16, 8, 16, 16, None, 0, 16, 8, 16, 16, 127, 0)
    with pytest.raises(ValueError, match="N must be"):
        ops.rms_norm_bwd_workspace_bytes(4, 40000)


def test_topk_distill_refusals():
    x, te, ix = t(4, 9), t(4, 3), t(4, 3, dtype=torch.int64)
    for err, match, args, kw in (
            (ValueError, r"logits must be a \(R, V\)", (t(9), te, ix), {}),
            (TypeError, "logits must be float32", (x.double(), te, ix), {}),
            (ValueError, "at least one column", (t(4, 0), te, ix), {}),
            (ValueError, r"teacher must be a \(R, K\)", (x, t(4), ix), {}),
            (ValueError, r"K must be in \[1, 512\]", (x, t(4, 0), t(4, 0, dtype=torch.int64)), {}),
            (ValueError, r"K must be in \[1, 512\]", (x, t(4, 513), t(4, 513, dtype=torch.int64)), {}),
            (ValueError, "teacher must have the shape", (x, t(5, 3), ix), {}),
            (TypeError, "teacher must be", (x, te.half(), ix), {}),
            (ValueError, "index must have the shape", (x, te, ix[:, :2]), {}),
            (TypeError, "index must be", (x, te, te), {}),
            (ValueError, "coef must have the shape", (x, te, ix), dict(coef=t(3))),
            (TypeError, "coef must be", (x, te, ix), dict(coef=t(4).half())),
            (ValueError, "temperature must be in", (x, te, ix), dict(temperature=0)),
            (ValueError, "temperature must be in", (x, te, ix), dict(temperature=float("nan"))),
            (ValueError, "temperature must be in", (x, te, ix), dict(temperature=float("inf"))),
            (ValueError, "no gradient is asked for", (x, te, ix), dict(grad=False, out=x)),
            (ValueError, "out must have the shape", (x, te, ix), dict(out=t(4, 8))),
            (TypeError, "out must be", (x, te, ix), dict(out=x.half())),
            (ValueError, "contiguous channels", (x, te, ix), dict(out=t(9, 4).t())),
            (TypeError, "logits must be a CUDA tensor", (x, te, ix), {})):
        with pytest.raises(err, match=match):
            sequence.topk_distill(*args, **kw)
    go = lambda **k: ops.topk_distill(*{**dict(  # noqa: E731
        dtype=1, tt=1, i64=1, R=4, V=9, K=3, logits=16, ldl=9, teacher=16, ldt=3, index=16, ldi=3, tau=1.0, coef=None, loss=16,
        d=32, ldd=9, ws=None, n=0, st=0), **k}.values())
    for match, kw in (("type must be", dict(dtype=4)), ("teacher's type", dict(tt=2)), (r"K in \[1, 512\]", dict(K=600)),
                      ("temperature must be", dict(tau=-1.0)), ("null pointer", dict(index=None)), ("overlap", dict(ldd=8)),
                      ("negative", dict(ldt=-3)), ("same row stride", dict(d=16, ldd=10)),
                      (r"workspace of \d+ bytes needed, 0 available", dict(V=300000, ldl=300000, ldd=300000))):
        with pytest.raises(ValueError, match=match):
            go(**kw)
    with pytest.raises(ValueError, match="bad type or sizes"):
        ops.topk_distill_workspace_bytes(1, 4, 0, 3)
    assert ops.topk_distill_workspace_bytes(1, 2048, 131072, 128) >= 0


def test_sizes_beyond_32_bits_are_refused():
    """Nothing is allocated: the rows are one, expanded."""
    many = 2 ** 32 + 4
    x, w = t(1, 8).expand(many, 8), t(8)
    for call in (lambda: sequence.rms_norm(x, w),
                 lambda: sequence.rms_norm_fp8(t(1, 8, dtype=torch.float16).expand(many, 8), w.half()),
                 lambda: sequence.rms_norm_backward(x, x, t(1).expand(many), w),
                 lambda: sequence.topk_distill(x, t(1, 3).expand(many, 3), t(1, 3, dtype=torch.int64).expand(many, 3)),
                 lambda: sequence.topk_distill(t(1, 1).expand(4, many), t(4, 3), t(4, 3, dtype=torch.int64)),
                 lambda: sequence.gated_scan_step(x, x, x), lambda: sequence.gated_scan(x[:, None], x[:, None]),
                 lambda: sequence.gated_scan(x[None], x[None])):
        with pytest.raises(ValueError, match="no size may be above"):
            call()
    with pytest.raises(ValueError, match="R in"):
        ops.rms_norm_fwd(1, 1, 1, 2 ** 31 - 1, 8, 16, 8, None, 0, 16, 1e-6, 16, 8, 0, None, None, 0, None, 0)
    with pytest.raises(ValueError, match="R in"):
        ops.rms_norm_bwd_workspace_bytes(2 ** 31 - 1, 8)
    with pytest.raises(ValueError, match="R in"):
        ops.topk_distill(1, 1, 1, 2 ** 31 - 1, 8, 3, 16, 8, 16, 3, 16, 3, 1.0, None, 16, None, 0, None, 0, 0)
