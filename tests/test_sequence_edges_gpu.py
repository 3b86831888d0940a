"""Edges of the operators of sequence policies (serl_amd/sequence.py): non-finite values, calls in place, strides and values at
the ends of their types, each against the operator's definition.  U, HALF and SMALL as in test_sequence_gpu.py."""
import math

import pytest
import torch

from test_sequence_gpu import norm_inputs, seq

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
