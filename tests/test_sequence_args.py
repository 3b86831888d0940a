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
    with pytest.raises(ValueError, match=r"workspace of \d+ bytes needed, 0 available"):
        scan(T=5000, gate_bs=40000, x_bs=40000, y_bs=40000)
    with pytest.raises(ValueError, match="bad type or sizes"):
        ops.gated_scan_workspace_bytes(9, 1, 1, 1)
    with pytest.raises(ValueError, match="bad sizes"):
        ops.gated_scan_states_floats(1, -1, 1)
    assert ops.gated_scan_workspace_bytes(1, 8, 4096, 2048) == 0
    assert ops.gated_scan_states_floats(2, 129, 8) == 2 * 2 * 8
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
