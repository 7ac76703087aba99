"""Operators on rows of class logits held on the device (torch CUDA tensors).

top_logits           a teacher's k largest logits a row, with the log-sum-exp of the rest
distill_loss         Kullback-Leibler loss of a student's rows against them
distill_derivatives  that loss with der1, its negative gradient
sample_classes       a class a row under temperature / top-k / top-p / min-p

Logits are [n, classes] tensors of 64, 32 or 16 bits (float16, bfloat16) with
any strides: `approx.t()` of a booster's dim-major [K, n] approximants is as
good as a row-major tensor.  Calls run on the tensor's device, on its current
torch stream, and do not wait; no autograd graph is recorded (der1 is the
derivative, with the sign of Derivatives.der1: minus the gradient).  Unlike
the rest of the package, which takes host arrays, these need torch.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Any, Optional

from . import _lib

MAX_CLASSES = 262144
MAX_TOP = 256

_torch = None  # and what is asked of it in every call, set by the first
_dtypes: dict = {}
_get_device = _get_stream = _L = None


def _t():
    global _torch, _get_device, _get_stream, _L
    if _torch is None:
        import torch
        _L = _lib.load()
        _dtypes.update({torch.float64: _lib.F64, torch.float32: _lib.F32, torch.float16: _lib.F16,
                        torch.bfloat16: _lib.BF16})
        if hasattr(torch._C, "_cuda_getCurrentRawStream"):
            # what torch.cuda.current_device and current_stream end in, without their objects
            _get_device, _get_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
        else:
            _get_device, _get_stream = torch.cuda.current_device, lambda d: torch.cuda.current_stream(d).cuda_stream
        _torch = torch
    return _torch


@dataclass
class TopLogits:
    """A teacher's rows: index [n, k] (int32 or int64; an index outside the
    classes is no entry, of equal indices in a row the first counts), value
    [n, k] logits, and tail [n], the log-sum-exp of the other classes at the
    temperature of the distillation (None: renormalised over the k)."""
    index: Any
    value: Any
    tail: Optional[Any] = None


@dataclass
class Distilled:
    """loss [n] and der1 [n, classes] = -d loss / d logits."""
    loss: Any
    der1: Any


def _bad(msg: str):
    return _lib.CbGpuError(_lib.ERR_INVALID, msg)


def _plain(who, name, x):
    # memory that stands for its negative (the imaginary part of a conjugate view) would be read as it is
    if x.is_neg():
        raise _bad(f"{who}: {name} is a negated view, pass {name}.resolve_neg()")


def _logits(who, x):
    torch = _torch or _t()
    if not isinstance(x, torch.Tensor):
        raise _bad(f"{who}: logits must be a torch tensor")
    shape = x.shape
    if len(shape) != 2:
        raise _bad(f"{who}: logits must be [n, classes], got {tuple(shape)}")
    dtype = _dtypes.get(x.dtype)
    if dtype is None:
        raise _bad(f"{who}: logits must be float64, float32, float16 or bfloat16, got {x.dtype}")
    n, V = shape
    if not 1 <= V <= MAX_CLASSES:
        raise _bad(f"{who}: {V} classes, outside 1..{MAX_CLASSES}")
    if n > 0x7fffffff:
        raise _bad(f"{who}: {n} rows, at most 2^31 - 1")
    _plain(who, "logits", x)
    if not x.is_cuda:
        raise _bad(f"{who}: logits must be on a CUDA device")
    rs, cs = x.stride()
    return _lib.Logits(x.data_ptr(), dtype, V, n, rs, cs)


def _side(who, name, v, x, shape, dtypes):
    """A contiguous operand beside the logits, of one of `dtypes`."""
    if not isinstance(v, _torch.Tensor) or v.get_device() != x.get_device():
        raise _bad(f"{who}: {name} must be a tensor on the logits' device")
    if v.dtype not in dtypes:
        raise _bad(f"{who}: {name} has dtype {v.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    if v.shape != shape:
        raise _bad(f"{who}: LengthMismatch: {name} is {tuple(v.shape)}, expected {shape}")
    _plain(who, name, v)
    return v if v.is_contiguous() else v.contiguous()


def _wide(x):
    return _torch.float64 if x.dtype == _torch.float64 else _torch.float32


def _run(x, fn, *args):
    """fn(*args, stream) on the device of x, on its current stream."""
    dev = x.get_device()
    if _get_device() == dev:
        rc = fn(*args, _get_stream(dev))
    else:
        with _torch.cuda.device(dev):
            rc = fn(*args, _get_stream(dev))
    if rc:
        _lib.check(rc)


def _temperature(who, t, least=1e-6):
    t = float(t)
    if not (least <= t <= 1e6 or (least == 0.0 and t == 0.0)) or (0.0 < t < 1e-6):
        raise _bad(f"{who}: temperature {t} is outside {'0 or ' if least == 0.0 else ''}1e-6..1e6")
    return t


def top_logits(logits, k: int, *, temperature: float = 1.0, tail: bool = True) -> TopLogits:
    """The k largest logits of every row in order (equal logits by lower
    index, NaN last), k up to min(256, classes): index int32 and value
    [n, k], and with `tail` the log-sum-exp [n] of the other classes at
    `temperature` (f64 for f64 logits, else f32)."""
    who = "top_logits"
    d = _logits(who, logits)
    k = int(k)
    if not 1 <= k <= min(MAX_TOP, d.n_classes):
        raise _bad(f"{who}: k = {k} is outside 1..min({MAX_TOP}, {d.n_classes} classes)")
    temperature = _temperature(who, temperature)
    n = d.n
    value = logits.new_empty(n, k)
    index = logits.new_empty(n, k, dtype=_torch.int32)
    rest = logits.new_empty(n, dtype=_wide(logits)) if tail else None
    _run(logits, _L.cbgpu_top_logits, C.byref(d), k, temperature, value.data_ptr(), index.data_ptr(),
         rest.data_ptr() if tail else None)
    return TopLogits(index, value, rest)


def _distill(who, logits, teacher, weight, temperature, der1, d=None):
    """The loss; der1, when not None, is checked unless `d`, the logits' description, comes with it."""
    own = d is not None
    if not own:
        d = _logits(who, logits)
    n = d.n
    wide = _wide(logits)
    if not isinstance(teacher, TopLogits):
        raise _bad(f"{who}: teacher must be a TopLogits")
    shape = getattr(teacher.index, "shape", ())
    if len(shape) != 2 or shape[0] != n or not 1 <= shape[1] <= MAX_TOP:
        raise _bad(f"{who}: LengthMismatch: the teacher's index is {tuple(shape)}, expected ({n}, 1..{MAX_TOP})")
    index = _side(who, "the teacher's index", teacher.index, logits, shape, (_torch.int32, _torch.int64))
    value = _side(who, "the teacher's value", teacher.value, logits, shape, tuple(_dtypes))
    rest = None if teacher.tail is None else _side(who, "the teacher's tail", teacher.tail, logits, (n,), (wide,))
    weight = None if weight is None else _side(who, "weight", weight, logits, (n,), (wide,))
    temperature = _temperature(who, temperature)
    if der1 is not None and not own:
        if not isinstance(der1, _torch.Tensor) or der1.get_device() != logits.get_device() or der1.dtype != logits.dtype:
            raise _bad(f"{who}: out must be a {logits.dtype} tensor on the logits' device")
        if der1.shape != logits.shape:
            raise _bad(f"{who}: LengthMismatch: out is {tuple(der1.shape)}, expected {tuple(logits.shape)}")
        _plain(who, "out", der1)
    loss = logits.new_empty(n, dtype=wide)
    t = _lib.Teacher(index.data_ptr(), value.data_ptr(), None if rest is None else rest.data_ptr(),
                     index.element_size(), _dtypes[value.dtype], shape[1])
    rs, cs = der1.stride() if der1 is not None else (0, 0)
    _run(logits, _L.cbgpu_distill, C.byref(d), C.byref(t), None if weight is None else weight.data_ptr(),
         temperature, loss.data_ptr(), None if der1 is None else der1.data_ptr(), rs, cs)
    return loss


def distill_loss(logits, teacher: TopLogits, *, weight=None, temperature: float = 1.0):
    """weight * T^2 * KL(teacher || student) of every row [n], over the
    teacher's classes and, with its tail, the bucket of all others.  A row of
    weight 0, of masked classes only or without a teacher's entry gives 0."""
    return _distill("distill_loss", logits, teacher, weight, temperature, None)


def distill_derivatives(logits, teacher: TopLogits, *, weight=None, temperature: float = 1.0,
                        out=None) -> Distilled:
    """distill_loss with der1 [n, classes], its negative derivative by the
    logits, in their dtype and layout.  `weight` is also the factor a caller's
    own loss puts on each row.  `out` takes der1; it may be the logits."""
    who = "distill_derivatives"
    if out is None:
        d = _logits(who, logits)
        dense = logits.is_contiguous() or (d.row_stride == 1 and d.class_stride == d.n)
        out = _torch.empty_like(logits) if dense else logits.new_empty(logits.shape)
        return Distilled(_distill(who, logits, teacher, weight, temperature, out, d), out)
    return Distilled(_distill(who, logits, teacher, weight, temperature, out), out)


def sample_classes(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One class a row [n] (int32) from softmax(logits / temperature), drawn by
    the given random numbers uniform [n] in [0, 1) (f32 or f64).

    In this order: top_k keeps the first k classes by logit (0: all); top_p
    keeps classes in order while the probability before them is below top_p
    of what top_k left; min_p keeps those of at least min_p times the largest
    probability.  Drawn is the first class by index whose running sum of kept
    probabilities exceeds uniform times their sum; temperature 0 gives the
    first class in order.  Each setting is a number or a tensor [n] (f32;
    top_k int32).  -1 for a row that holds a NaN or masks every class."""
    who = "sample_classes"
    d = _logits(who, logits)
    n = d.n
    f32 = _torch.float32
    u = _side(who, "uniform", uniform, logits, (n,), (f32, _torch.float64))
    keep = [u]

    def rows(name, v, dtype):
        if not isinstance(v, _torch.Tensor):
            return None
        keep.append(_side(who, name, v, logits, (n,), (dtype,)))
        return keep[-1].data_ptr()

    s = _lib.Sampling(u.data_ptr(), rows("temperature", temperature, f32), rows("top_p", top_p, f32),
                      rows("min_p", min_p, f32), rows("top_k", top_k, _torch.int32))
    s.uniform_dtype = _dtypes[u.dtype]
    if s.temperature_rows is None:
        s.temperature = _temperature(who, temperature, 0.0)
    if s.top_p_rows is None:
        s.top_p = float(top_p)
        if not 0.0 <= s.top_p <= 1.0:
            raise _bad(f"{who}: top_p {top_p} is outside 0..1")
    if s.min_p_rows is None:
        s.min_p = float(min_p)
        if not 0.0 <= s.min_p <= 1.0:
            raise _bad(f"{who}: min_p {min_p} is outside 0..1")
    if s.top_k_rows is None:
        if int(top_k) < 0:
            raise _bad(f"{who}: top_k {top_k} < 0")
        s.top_k = min(int(top_k), MAX_CLASSES)
    index = logits.new_empty(n, dtype=_torch.int32)
    _run(logits, _L.cbgpu_sample_classes, C.byref(d), C.byref(s), index.data_ptr())
    return index
