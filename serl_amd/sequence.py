"""Operators of sequence policies on CUDA tensors: a gated linear recurrence (the memory), the root-mean-square norm with
the residual's addition, and the distillation of a teacher's top logits -- each with its gradient, all arithmetic in HIP
kernels (csrc/gated_scan.hip, rms_norm.hip, distill.hip).  No counterpart in the reference: its policies see history
through frame stacks (serl/networks/pixel_multiplexer.py:27) and its only discrete head is the gripper's
(serl/agents/bc/pixel_hybrid_bc_learner.py).

Tensors are float32, bfloat16 or float16 on one GPU, channels contiguous (others are copied first); states, statistics and
sums are float32 and a value is rounded once, when it is stored.  Calls are enqueued on the current stream of the tensors'
device, wait for nothing, and may be captured into a graph; results and scratch memory come from torch's allocator, call by
call, so nothing is shared between calls or graphs.  As in the learners, gradients are explicit calls: autograd records
nothing here, and the gradient of an expanded (broadcast) input comes full size, for the caller to sum.  Wrong types raise
TypeError, wrong shapes ValueError, before anything is enqueued.  The same arguments, laid out the same, give the same bits
on every call."""
from __future__ import annotations

import contextlib
import functools

import torch

from . import ops

_CODES = {torch.float32: ops.F32, torch.bfloat16: ops.BF16, torch.float16: ops.F16}
_NO_GUARD = contextlib.nullcontext()
_ROWS = torch.contiguous_format
try:                                    # the handle alone: a tenth of the time of torch.cuda.current_stream(), which makes an object
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:
    def _raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream
try:                                    # the tensors at hand have initialised the GPU: without torch.cuda's question whether it is
    _device = torch._C._cuda_getDevice
except AttributeError:
    _device = torch.cuda.current_device
# scratch sizes depend on the calls' sizes alone
_scan_bytes = functools.lru_cache(1024)(ops.gated_scan_workspace_bytes)
_norm_bytes = functools.lru_cache(1024)(ops.rms_norm_bwd_workspace_bytes)
_distill_bytes = functools.lru_cache(1024)(ops.topk_distill_workspace_bytes)


def _shape(t, name, shape):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.shape != shape:
        raise ValueError(f"{name} must have the shape {tuple(shape)}, got {tuple(t.shape)}")


_MOST = 0x7fff0000                      # sizes are 32-bit integers in the C ABI, which would cut them


def _sizes(*n):
    if max(n) > _MOST:
        raise ValueError(f"no size may be above {_MOST}, got {max(n)}")


def _type(t, name, *dtypes):
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")


def _place(names, *tensors):
    """The tensors' common GPU: the context that makes it the current one."""
    at = None
    for i, t in enumerate(tensors):
        if t is None:
            continue
        d = t.get_device()              # -1: not on a GPU
        if d < 0:
            raise TypeError(f"{names[i]} must be a CUDA tensor")
        if at is None:
            at = d
        elif d != at:
            raise ValueError(f"{names[i]} is on {t.device}, the others on cuda:{at}")
    return _NO_GUARD if at == _device() else torch.cuda.device(at)


def _channels(t):
    """t with contiguous channels (the last dimension)."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _out(t, name, like_shape, dtype):
    """A caller's output tensor: rows may have any stride, but must not share memory with each other."""
    _shape(t, name, like_shape)
    _type(t, name, dtype)
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} must have contiguous channels")
    return t


# ------------------------------------------------------------------------------------------------- gated recurrence
def _scan_args(gate, x, starts, lengths):
    if not isinstance(gate, torch.Tensor) or gate.ndim != 3:
        raise ValueError("gate must be a (B, T, D) tensor")
    B, T, D = gate.shape
    _sizes(B, T, D)
    _shape(x, "x", (B, T, D))
    if gate.dtype not in _CODES:
        raise TypeError(f"gate must be float32, bfloat16 or float16, got {gate.dtype}")
    _type(x, "x", gate.dtype)
    if starts is not None:
        _shape(starts, "starts", (B, T))
        _type(starts, "starts", torch.bool, torch.uint8)
    if lengths is not None:
        _shape(lengths, "lengths", (B,))
        _type(lengths, "lengths", torch.int32, torch.int64)
    return B, T, D


def _state(t, name, B, D):
    if t is not None:
        _shape(t, name, (B, D))
        _type(t, name, torch.float32)


def _masks(starts, lengths, T):
    if starts is not None:
        starts = _channels(starts)
    if lengths is not None:
        if lengths.dtype == torch.int64:
            lengths = lengths.clamp(0, T).to(torch.int32)
        lengths = lengths.contiguous()
    return starts, lengths


def _scan_scratch(code, B, T, D, device):
    n = _scan_bytes(code, B, T, D)
    return (torch.empty(n // 4, dtype=torch.float32, device=device) if n else None), n


def gated_scan(gate, x, h0=None, starts=None, lengths=None, save=False):
    """h_t = f_t (starts_t ? 0 : h_{t-1}) + (1 - f_t) x_t with f = sigmoid(gate), along the time axis.

    gate, x: (B, T, D); h0: (B, D) float32 state before the first step (None: zeros); starts: (B, T) bool, an episode
    begins at the step; lengths: (B,) ints, steps from there on hold the state and give y = 0.  T and B may be 0.
    An infinity or NaN in the state stays in its channel until an episode begins.
    Returns (y, h_last): y (B, T, D) in gate's type, h_last (B, D) float32; with save=True also the states that
    gated_scan_backward needs."""
    B, T, D = _scan_args(gate, x, starts, lengths)
    _state(h0, "h0", B, D)
    with _place(("gate", "x", "h0", "starts", "lengths"), gate, x, h0, starts, lengths):
        gate, x = _channels(gate), _channels(x)
        starts, lengths = _masks(starts, lengths, T)
        if h0 is not None:
            h0 = h0.contiguous()
        code, dev = _CODES[gate.dtype], gate.device
        y = torch.empty_like(gate, memory_format=_ROWS)
        h_last = gate.new_empty((B, D), dtype=torch.float32)
        saved = gate.new_empty((B, -(-T // 64), D), dtype=torch.float32) if save else None
        ws, nws = _scan_scratch(code, B, T, D, dev)
        ops.gated_scan_fwd(code, B, T, D, gate.data_ptr(), gate.stride(0), gate.stride(1), x.data_ptr(), x.stride(0),
                           x.stride(1), _ptr(h0), _ptr(starts), 0 if starts is None else starts.stride(0), _ptr(lengths),
                           y.data_ptr(), T * D, D, h_last.data_ptr(), _ptr(saved), _ptr(ws), nws, _raw_stream(dev.index))
    return (y, h_last, saved) if save else (y, h_last)


def gated_scan_backward(gate, x, saved, dy, dh_last=None, starts=None, lengths=None, out=None):
    """Gradients of gated_scan: (dgate, dx) in gate's type, dh0 (B, D) float32.  `saved` and the other arguments as in the
    forward call; dy (B, T, D), dh_last (B, D) float32 or None.  out: (dgate, dx) tensors to write, for instance the two
    halves of one projection's gradient; they share no memory with each other or the inputs."""
    B, T, D = _scan_args(gate, x, starts, lengths)
    _shape(saved, "saved", (B, -(-T // 64), D))
    _type(saved, "saved", torch.float32)
    _shape(dy, "dy", (B, T, D))
    _type(dy, "dy", gate.dtype)
    _state(dh_last, "dh_last", B, D)
    if out is not None:
        dgate, dx = _out(out[0], "out[0]", (B, T, D), gate.dtype), _out(out[1], "out[1]", (B, T, D), gate.dtype)
    else:
        dgate = dx = None
    with _place(("gate", "x", "saved", "dy", "dh_last", "starts", "lengths", "out[0]", "out[1]"), gate, x, saved, dy, dh_last,
                starts, lengths, dgate, dx):
        gate, x, dy, saved = _channels(gate), _channels(x), _channels(dy), saved.contiguous()
        starts, lengths = _masks(starts, lengths, T)
        if dh_last is not None:
            dh_last = dh_last.contiguous()
        code, dev = _CODES[gate.dtype], gate.device
        if out is None:
            dgate, dx = torch.empty_like(gate, memory_format=_ROWS), torch.empty_like(gate, memory_format=_ROWS)
        if T == 0:
            dh0 = torch.zeros((B, D), dtype=torch.float32, device=dev) if dh_last is None else dh_last.clone()
            return dgate, dx, dh0
        dh0 = gate.new_empty((B, D), dtype=torch.float32)
        ws, nws = _scan_scratch(code, B, T, D, dev)
        ops.gated_scan_bwd(code, B, T, D, gate.data_ptr(), gate.stride(0), gate.stride(1), x.data_ptr(), x.stride(0),
                           x.stride(1), _ptr(starts), 0 if starts is None else starts.stride(0), _ptr(lengths),
                           saved.data_ptr(), dy.data_ptr(), dy.stride(0), dy.stride(1), _ptr(dh_last), dgate.data_ptr(),
                           dgate.stride(0), dgate.stride(1), dx.data_ptr(), dx.stride(0), dx.stride(1), dh0.data_ptr(),
                           _ptr(ws), nws, _raw_stream(dev.index))
    return dgate, dx, dh0


def gated_scan_step(gate, x, h, starts=None, h_out=None):
    """One step of gated_scan for an acting policy: gate, x (B, D), state h (B, D) float32, starts (B,) bool or None.
    Returns (y, h_new); h_out: the tensor to write the new state to (h itself: in place)."""
    if not isinstance(gate, torch.Tensor) or gate.ndim != 2:
        raise ValueError("gate must be a (B, D) tensor")
    B, D = gate.shape
    _sizes(B, D)
    _shape(x, "x", (B, D))
    if gate.dtype not in _CODES:
        raise TypeError(f"gate must be float32, bfloat16 or float16, got {gate.dtype}")
    _type(x, "x", gate.dtype)
    if h is None:
        raise TypeError("h must be a tensor")
    _state(h, "h", B, D)
    if starts is not None:
        _shape(starts, "starts", (B,))
        _type(starts, "starts", torch.bool, torch.uint8)
    if h_out is not None:
        _state(h_out, "h_out", B, D)
        if not h_out.is_contiguous():
            raise ValueError("h_out must be contiguous")
    with _place(("gate", "x", "h", "starts", "h_out"), gate, x, h, starts, h_out):
        gate, x, h = _channels(gate), _channels(x), h.contiguous()
        y = torch.empty_like(gate, memory_format=_ROWS)
        if h_out is None:
            h_out = torch.empty_like(h, memory_format=_ROWS)
        ops.gated_scan_fwd(_CODES[gate.dtype], B, 1, D, gate.data_ptr(), gate.stride(0), 0, x.data_ptr(), x.stride(0), 0,
                           h.data_ptr(), _ptr(starts), 0 if starts is None else starts.stride(0), None, y.data_ptr(), D, D,
                           h_out.data_ptr(), None, None, 0, _raw_stream(gate.device.index))
    return y, h_out


# --------------------------------------------------------------------------------- root-mean-square norm + residual
def _rows(t):
    """t as (R, N) rows with contiguous channels (a view wherever its strides allow one)."""
    t = _channels(t)
    return t if t.ndim == 2 else t.reshape(-1, t.shape[-1])


def _width(t, name):
    if not isinstance(t, torch.Tensor) or t.ndim < 1:
        raise ValueError(f"{name} must be a (..., N) tensor")
    if not 1 <= t.shape[-1] <= 32768:
        raise ValueError(f"{name}: N must be in [1, 32768], got {t.shape[-1]}")
    _sizes(t.numel() // t.shape[-1])


def _norm_args(x, weight, residual):
    _width(x, "x")
    if x.dtype not in _CODES:
        raise TypeError(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    _shape(weight, "weight", (x.shape[-1],))
    _type(weight, "weight", x.dtype, torch.float32)
    if residual is not None:
        _shape(residual, "residual", x.shape)
        _type(residual, "residual", x.dtype, torch.float32)


def _norm(x, weight, residual, eps, fp8, save):
    _norm_args(x, weight, residual)
    with _place(("x", "weight", "residual"), x, weight, residual):
        shape, N = x.shape, x.shape[-1]
        rows, res, weight = _rows(x), None if residual is None else _rows(residual), weight.contiguous()
        R, dev = rows.shape[0], x.device
        y = torch.empty_like(x, dtype=torch.float8_e4m3fn if fp8 else x.dtype, memory_format=_ROWS)
        scale = x.new_empty(shape[:-1], dtype=torch.float32) if fp8 else None
        total = x if res is None else torch.empty_like(residual, memory_format=_ROWS)
        rstd = x.new_empty(shape[:-1], dtype=torch.float32) if save else None
        code = _CODES[x.dtype]
        ops.rms_norm_fwd(code, code if res is None else _CODES[residual.dtype], _CODES[weight.dtype], R, N, rows.data_ptr(),
                         rows.stride(0), _ptr(res), 0 if res is None else res.stride(0), weight.data_ptr(), eps, y.data_ptr(),
                         N, fp8, _ptr(scale), None if res is None else total.data_ptr(), N, _ptr(rstd), _raw_stream(dev.index))
    return y, scale, total, rstd


def rms_norm(x, weight, residual=None, eps=1e-6, save=False):
    """y = s / sqrt(mean(s^2) + eps) * weight over the last dimension (1 .. 32768), s = x + residual.

    residual: x's shape, in x's type or float32 (a residual stream kept in 32 bits); weight (N,) in x's type or float32.
    The squares are summed in float32: a row with values beyond some 1e19 gives y = 0.
    Returns (y, s): y in x's type, s in the residual's (rounded to it before it is normed), or x itself without a residual;
    with save=True also rstd (...,) float32 for rms_norm_backward."""
    y, _, total, rstd = _norm(x, weight, residual, eps, False, save)
    return (y, total, rstd) if save else (y, total)


def rms_norm_fp8(x, weight, residual=None, eps=1e-6):
    """rms_norm with its output in 8 bits: (q, scale, s), q float8_e4m3fn and scale (...,) float32 per row such that
    y = q * scale; scale = max(|y|) / 448, at least 2^-126, and 1 for a row of zeros.  A row that holds a NaN has the
    scale NaN."""
    y, scale, total, _ = _norm(x, weight, residual, eps, True, False)
    return y, scale, total


def rms_norm_backward(dy, s, rstd, weight, ds=None):
    """Gradients of rms_norm: (dx, dweight).  s and rstd as the forward call returned them; dy in the type of its x; ds: the
    gradient that reaches s itself (the residual stream behind), in s's type.  dx, in s's type, is the gradient of x and of
    the residual alike; dweight (N,) float32."""
    _width(s, "s")
    _shape(dy, "dy", s.shape)
    if dy.dtype not in _CODES:
        raise TypeError(f"dy must be float32, bfloat16 or float16, got {dy.dtype}")
    _type(s, "s", dy.dtype, torch.float32)
    _shape(rstd, "rstd", s.shape[:-1])
    _type(rstd, "rstd", torch.float32)
    _shape(weight, "weight", (s.shape[-1],))
    _type(weight, "weight", dy.dtype, torch.float32)
    if ds is not None:
        _shape(ds, "ds", s.shape)
        _type(ds, "ds", s.dtype)
    with _place(("s", "dy", "rstd", "weight", "ds"), s, dy, rstd, weight, ds):
        N = s.shape[-1]
        sr, yr, dr = _rows(s), _rows(dy), None if ds is None else _rows(ds)
        weight, rstd = weight.contiguous(), rstd.contiguous()
        R, dev = sr.shape[0], s.device
        dx = torch.empty_like(s, memory_format=_ROWS)
        dw = s.new_empty(N, dtype=torch.float32)
        n = _norm_bytes(R, N)
        ws = torch.empty(n // 4, dtype=torch.float32, device=dev) if n else None
        ops.rms_norm_bwd(_CODES[dy.dtype], _CODES[s.dtype], _CODES[weight.dtype], R, N, yr.data_ptr(), yr.stride(0),
                         sr.data_ptr(), sr.stride(0), rstd.data_ptr(), weight.data_ptr(), _ptr(dr),
                         0 if dr is None else dr.stride(0), dx.data_ptr(), N, dw.data_ptr(), _ptr(ws), n,
                         _raw_stream(dev.index))
    return dx, dw


# ------------------------------------------------------------------------------ distillation from a teacher's top logits
def topk_distill(logits, teacher, index, temperature=1.0, coef=None, grad=True, out=None):
    """loss_r = coef_r T^2 KL(q || p), q = softmax(teacher / T) over a row's K slots, p = softmax(logits / T) over its V
    columns, and its gradient with respect to the logits, coef_r T (p - q), in one pass over them.

    logits: (R, V); teacher: (R, K) logits in logits' type or float32, 1 <= K <= 512; index: (R, K) int64 or int32 columns of
    them; coef: (R,) float32 weights (None: ones).  A slot is absent if its index is outside [0, V) or its logit -inf; a row
    without slots, or with coef 0, gives loss 0 and gradient 0 whatever it holds.  A column named twice gets both shares.
    Returns (loss (R,) float32, dlogits in logits' type), dlogits None with grad=False; out: the tensor for dlogits, which may
    be logits itself."""
    if not isinstance(logits, torch.Tensor) or logits.ndim != 2:
        raise ValueError("logits must be a (R, V) tensor")
    if logits.dtype not in _CODES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    R, V = logits.shape
    _sizes(R, V)
    if V < 1:
        raise ValueError("logits must have at least one column")
    if not isinstance(teacher, torch.Tensor) or teacher.ndim != 2:
        raise ValueError("teacher must be a (R, K) tensor")
    K = teacher.shape[1]
    if not 1 <= K <= 512:
        raise ValueError(f"teacher: K must be in [1, 512], got {K}")
    _shape(teacher, "teacher", (R, K))
    _type(teacher, "teacher", logits.dtype, torch.float32)
    _shape(index, "index", (R, K))
    _type(index, "index", torch.int64, torch.int32)
    if coef is not None:
        _shape(coef, "coef", (R,))
        _type(coef, "coef", torch.float32)
    temperature = float(temperature)
    if not 2.0 ** -20 <= temperature <= 2.0 ** 20:
        raise ValueError(f"temperature must be in [2^-20, 2^20], got {temperature}")
    if out is not None:
        if not grad:
            raise ValueError("out is given, but no gradient is asked for")
        _out(out, "out", (R, V), logits.dtype)
    with _place(("logits", "teacher", "index", "coef", "out"), logits, teacher, index, coef, out):
        logits = _channels(logits)
        teacher, index = _channels(teacher), _channels(index)
        if coef is not None:
            coef = coef.contiguous()
        dev, code = logits.device, _CODES[logits.dtype]
        loss = logits.new_empty(R, dtype=torch.float32)
        if grad and out is None:
            out = torch.empty_like(logits, memory_format=_ROWS)
        n = _distill_bytes(code, R, V, K)
        ws = torch.empty(n // 4, dtype=torch.float32, device=dev) if n else None
        ops.topk_distill(code, _CODES[teacher.dtype], index.dtype == torch.int64, R, V, K, logits.data_ptr(), logits.stride(0),
                         teacher.data_ptr(), teacher.stride(0), index.data_ptr(), index.stride(0), temperature, _ptr(coef),
                         loss.data_ptr(), _ptr(out), 0 if out is None else out.stride(0), _ptr(ws), n, _raw_stream(dev.index))
    return loss, out
