"""Distributions over classes -- the disparity bins of a volume, or any other soft-max axis -- as HIP
kernels: scoring (log-probability of a given class, entropy, top alternatives) and distillation from
a teacher known by its top entries, both differentiable.

They stand next to the disparity regression of `disparity.soft_argmin` (the reference's
/root/reference/model/model.py:417-429, 454-456; the reference itself has neither operator):

    teacher = log_probs(teacher_cost, scale=-1.0, top=8)                    # 64 bytes a pixel instead of 4 D
    loss = distill_loss(student_cost, teacher.top_log_prob, teacher.top_index, scale=-1.0)   # (B, H, W)
    nll = -log_probs(student_cost, true_bin, scale=-1.0).log_prob           # 0 where true_bin is no bin
    (loss + nll).mean().backward()

Logits are float32, bfloat16 or float16; the class axis is `dim` (1, as in a (B, D, H, W) volume or a
(rows, classes) matrix), and `scale * logits` are the log-weights: -1 for a cost volume, 1/T for a
temperature.  Tensors in memory order, or with the class axis last in memory (torch's channels_last),
are read where they are; any other order is copied first.  Sums and results are float32, gradients
have the type and the memory order of the logits.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["LogProbs", "log_probs", "distill_loss"]

_DTYPES = {torch.float32: _lib.DW_DTYPE_F32, torch.bfloat16: _lib.DW_DTYPE_BF16, torch.float16: _lib.DW_DTYPE_F16}
_TEACHER_FLAGS = {torch.float32: 0, torch.bfloat16: _lib.DW_DIST_TEACHER_BF16, torch.float16: _lib.DW_DIST_TEACHER_F16}
_INDEX_FLAGS = {torch.int32: 0, torch.int64: _lib.DW_DIST_INDEX64}


class LogProbs(NamedTuple):
    log_prob: Optional[Tensor]   # of the given class; 0 where none is given; None without an index
    entropy: Tensor              # of the row's distribution, in nats
    top_log_prob: Tensor         # the `top` most likely classes along the class axis, descending
    top_index: Tensor            # their indices, int32; ties: the lowest first


@functools.lru_cache(maxsize=1024)
def _desc(workspace_of, outer, classes, inner, stride, scale, dtype, entries, flags):
    """(descriptor for ctypes, workspace bytes) of one problem; raises on what the library refuses."""
    d = _lib.DwDistDesc(outer, classes, inner, stride, scale, dtype, entries, flags)
    ref = C.byref(d)
    nbytes = getattr(_lib.lib(), workspace_of)(ref)
    if nbytes < 0:
        _lib.check(int(nbytes), f"{workspace_of}(classes={classes}, entries={entries}, scale={scale})")
    return ref, nbytes


def _place(x: Tensor, dim: int) -> Tuple[Tensor, int]:
    """The tensor as the kernels read it, and DW_DIST_LAST if its classes lie together."""
    if x.is_contiguous():
        return x, 0
    if x.movedim(dim, -1).is_contiguous():
        return x, _lib.DW_DIST_LAST
    return x.contiguous(), 0


def _sizes(x: Tensor, dim: int) -> Tuple[int, int, int]:
    return math.prod(x.shape[:dim]), x.shape[dim], math.prod(x.shape[dim + 1:])


def _rows_shape(x: Tensor, dim: int):
    return x.shape[:dim] + x.shape[dim + 1:]


# Host time counts: a small training step is bound by it, and the interpreter runs cold in the autograd
# engine's own thread.  So the backward passes find their descriptor made, and the device and stream are
# read without building torch.cuda.Stream objects where torch has the calls its own compiler uses.
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(device: torch.device, name: str, *args) -> None:
    """One library call on the device's current stream (the library launches on the current device)."""
    index = device.index
    if _current_device() == index:
        rc = getattr(_lib.lib(), name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = getattr(_lib.lib(), name)(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


def _ptr(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


def _workspace(x: Tensor, nbytes: int) -> Optional[Tensor]:
    # allocated for each call: calls on other streams, or captured into other graphs, have their own
    return torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None


# ------------------------------------------------------------------------------ log-probabilities

def _lp_desc(x: Tensor, last: int, index: Optional[Tensor], dim: int, scale: float, top: int):
    outer, V, inner = _sizes(x, dim)
    flags = last if index is None else last | _INDEX_FLAGS[index.dtype]
    return _desc("dw_log_probs_workspace_bytes", outer, V, inner, (0, 0, 0), scale, _DTYPES[x.dtype], top, flags)


def _lp_forward(x: Tensor, last: int, index: Optional[Tensor], dim: int, top: int, need_stats: bool, ref, nbytes: int):
    rows = _rows_shape(x, dim)
    dev = x.device
    ent = torch.empty(rows, dtype=torch.float32, device=dev)
    lp = torch.empty_like(ent) if index is not None else torch.empty((0,), dtype=torch.float32, device=dev)
    stats = torch.empty(rows + (3,), dtype=torch.float32, device=dev) if need_stats else None
    if last:   # the kernels write the list of a row together, too
        top_lp = torch.empty(rows + (top,), dtype=torch.float32, device=dev).movedim(-1, dim)
        top_idx = torch.empty(rows + (top,), dtype=torch.int32, device=dev).movedim(-1, dim)
    else:
        shape = x.shape[:dim] + (top,) + x.shape[dim + 1:]
        top_lp = torch.empty(shape, dtype=torch.float32, device=dev)
        top_idx = torch.empty(shape, dtype=torch.int32, device=dev)
    ws = _workspace(x, nbytes)
    _call(dev, "dw_log_probs_fwd", ref, x.data_ptr(), _ptr(index), lp.data_ptr() if index is not None else None,
          ent.data_ptr(), top_lp.data_ptr() if top else None, top_idx.data_ptr() if top else None, _ptr(stats),
          _ptr(ws), nbytes)
    return lp, ent, top_lp, top_idx, stats


def _lp_backward(x: Tensor, index: Optional[Tensor], stats: Tensor, g_lp: Optional[Tensor], g_ent: Optional[Tensor],
                 ref) -> Tensor:
    grad = torch.empty_like(x)
    if g_lp is not None:
        g_lp = g_lp.contiguous() if index is not None else None
    if g_ent is not None:
        g_ent = g_ent.contiguous()
    _call(x.device, "dw_log_probs_bwd", ref, x.data_ptr(), _ptr(index), stats.data_ptr(), _ptr(g_lp), _ptr(g_ent),
          grad.data_ptr())
    return grad


def _once(backward):
    """`once_differentiable`, whose bookkeeping only a pass that builds a graph has to pay for."""
    guarded = once_differentiable(backward)
    return lambda ctx, *grads: (guarded if torch.is_grad_enabled() else backward)(ctx, *grads)


def _lp_node_backward(ctx, g_lp, g_ent, _g_top, _g_index):
    logits, index = ctx.saved_tensors
    if g_lp is None and g_ent is None:
        return None, None, None, None, None
    x = logits if ctx.in_place else logits.contiguous()
    return _lp_backward(x, index, ctx.stats, g_lp, g_ent, ctx.ref), None, None, None, None


class _LogProbsFunction(torch.autograd.Function):
    """Eager calls with a gradient skip the operator dispatcher."""

    @staticmethod
    def forward(ctx, logits, index, dim, scale, top):
        x, last = _place(logits, dim)
        ctx.ref, nbytes = _lp_desc(x, last, index, dim, scale, top)
        lp, ent, top_lp, top_idx, ctx.stats = _lp_forward(x, last, index, dim, top, True, ctx.ref, nbytes)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(top_lp, top_idx)
        ctx.save_for_backward(logits, index)
        ctx.in_place = x is logits
        return lp, ent, top_lp, top_idx

    backward = staticmethod(_once(_lp_node_backward))


@torch.library.custom_op("depthwarp::log_probs", mutates_args=())
def _log_probs_op(logits: Tensor, index: Optional[Tensor], dim: int, scale: float,
                  top: int) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """The same as a torch operator (what torch.compile traces); the last result is the backward's."""
    x, last = _place(logits, dim)
    index = None if index is None else index.contiguous()
    return _lp_forward(x, last, index, dim, top, True, *_lp_desc(x, last, index, dim, scale, top))


@_log_probs_op.register_fake
def _(logits, index, dim, scale, top):
    x, last = _place(logits, dim)
    rows = _rows_shape(x, dim)
    ent = x.new_empty(rows, dtype=torch.float32)
    lp = torch.empty_like(ent) if index is not None else x.new_empty((0,), dtype=torch.float32)
    if last:
        top_lp = x.new_empty(rows + (top,), dtype=torch.float32).movedim(-1, dim)
        top_idx = x.new_empty(rows + (top,), dtype=torch.int32).movedim(-1, dim)
    else:
        shape = x.shape[:dim] + (top,) + x.shape[dim + 1:]
        top_lp, top_idx = x.new_empty(shape, dtype=torch.float32), x.new_empty(shape, dtype=torch.int32)
    return lp, ent, top_lp, top_idx, x.new_empty(rows + (3,), dtype=torch.float32)


@torch.library.custom_op("depthwarp::log_probs_bwd", mutates_args=())
def _log_probs_bwd_op(logits: Tensor, index: Optional[Tensor], stats: Tensor, g_lp: Optional[Tensor],
                      g_ent: Optional[Tensor], dim: int, scale: float) -> Tensor:
    x, last = _place(logits, dim)
    index = None if index is None else index.contiguous()
    return _lp_backward(x, index, stats, g_lp, g_ent, _lp_desc(x, last, index, dim, scale, 0)[0])


@_log_probs_bwd_op.register_fake
def _(logits, index, stats, g_lp, g_ent, dim, scale):
    return torch.empty_like(_place(logits, dim)[0])


def _lp_setup(ctx, inputs, output):
    logits, index, dim, scale, _top = inputs
    ctx.mark_non_differentiable(*output[2:])
    ctx.save_for_backward(logits, index, output[4])
    ctx.dim, ctx.scale = dim, scale


def _lp_op_backward(ctx, g_lp, g_ent, _g_top, _g_index, _g_stats):
    logits, index, stats = ctx.saved_tensors
    return _log_probs_bwd_op(logits, index, stats, g_lp, g_ent, ctx.dim, ctx.scale), None, None, None, None


_log_probs_op.register_autograd(_lp_op_backward, setup_context=_lp_setup)


def _check_logits(logits: Tensor, dim: int, scale: float) -> Tuple[int, float]:
    if not logits.is_cuda:
        raise _lib.DepthwarpError(f"logits: expected a ROCm device tensor, got {logits.device} "
                                  "(the HIP kernels have no CPU path)")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits: expected float32, bfloat16 or float16, got {logits.dtype}")
    n = logits.dim()
    if not -n <= dim < n:
        raise ValueError(f"dim: no axis {dim} in logits of shape {tuple(logits.shape)}")
    dim %= n
    if logits.shape[dim] == 0:
        raise ValueError(f"logits: no classes along axis {dim} of {tuple(logits.shape)}")
    scale = float(scale)
    if not math.isfinite(scale) or scale == 0.0:
        raise ValueError(f"scale: expected a finite number other than 0, got {scale}")
    return dim, scale


def _check_index(name: str, index: Tensor, shape, device) -> None:
    if index.dtype not in _INDEX_FLAGS:
        raise TypeError(f"{name}: expected int32 or int64, got {index.dtype}")
    if index.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(index.shape)}")
    if index.device != device:
        raise ValueError(f"{name}: expected a tensor on {device}, got {index.device}")


def log_probs(logits: Tensor, index: Optional[Tensor] = None, *, dim: int = 1, scale: float = 1.0,
              top: int = 0) -> LogProbs:
    """Scores rows of `logits` against the classes `index` and describes their distribution.

    `index` (int32 or int64) has the shape of `logits` without `dim`; a value outside [0, classes) means
    that no class is given there (a pixel without ground truth, or beyond the range): log-probability 0 and
    no gradient.  `top` (0 to 64) most likely classes come back as log-probabilities and int32 indices, in
    descending order, equal values by lowest index.

    `log_prob` and `entropy` are differentiable with respect to `logits`, once; the top lists are not.
    A class at -inf has probability 0; a row of nothing else has entropy 0, log-probability -inf and
    gradient 0.  A row with NaN (or +inf) has NaN results.  A row that gets no upstream gradient gets
    zeros whatever it holds.
    """
    dim, scale = _check_logits(logits, dim, scale)
    top = int(top)
    if not 0 <= top <= min(_lib.DW_DIST_MAX_ENTRIES, logits.shape[dim]):
        raise ValueError(f"top: expected 0 to {min(_lib.DW_DIST_MAX_ENTRIES, logits.shape[dim])}, got {top}")
    if index is not None:
        _check_index("index", index, _rows_shape(logits, dim), logits.device)
        index = index.contiguous()
    if torch.compiler.is_compiling():
        lp, ent, top_lp, top_idx, _ = _log_probs_op(logits, index, dim, scale, top)
    elif logits.requires_grad and torch.is_grad_enabled():
        lp, ent, top_lp, top_idx = _LogProbsFunction.apply(logits, index, dim, scale, top)
    else:
        x, last = _place(logits, dim)
        lp, ent, top_lp, top_idx, _ = _lp_forward(x, last, index, dim, top, False,
                                                  *_lp_desc(x, last, index, dim, scale, top))
    return LogProbs(lp if index is not None else None, ent, top_lp, top_idx)


# --------------------------------------------------------------------------------- distillation

def _entries(teacher: Tensor, index: Tensor, dim: int):
    """The list's two tensors in one memory order, and its element strides along outer, entry, inner."""
    if not (teacher.is_contiguous() and index.is_contiguous()):
        if teacher.movedim(dim, -1).is_contiguous() and index.movedim(dim, -1).is_contiguous():
            _, k, inner = _sizes(teacher, dim)
            return teacher, index, (k * inner, 1, k)
        teacher, index = teacher.contiguous(), index.contiguous()
    _, k, inner = _sizes(teacher, dim)
    return teacher, index, (k * inner, inner, 1)


def _ds_desc(logits: Tensor, teacher: Tensor, index: Tensor, dim: int, scale: float, renormalise: bool):
    x, last = _place(logits, dim)
    teacher, index, stride = _entries(teacher, index, dim)
    outer, V, inner = _sizes(x, dim)
    flags = last | _INDEX_FLAGS[index.dtype] | _TEACHER_FLAGS[teacher.dtype]
    if renormalise:
        flags |= _lib.DW_DIST_RENORMALISE
    return x, teacher, index, _desc("dw_distill_workspace_bytes", outer, V, inner, stride, scale, _DTYPES[x.dtype],
                                    teacher.shape[dim], flags)


def _ds_forward(x: Tensor, teacher: Tensor, index: Tensor, dim: int, need_stats: bool, ref, nbytes: int):
    rows = _rows_shape(x, dim)
    loss = torch.empty(rows, dtype=torch.float32, device=x.device)
    stats = torch.empty(rows + (4,), dtype=torch.float32, device=x.device) if need_stats else None
    ws = _workspace(x, nbytes)
    _call(x.device, "dw_distill_fwd", ref, x.data_ptr(), teacher.data_ptr(), index.data_ptr(), loss.data_ptr(),
          _ptr(stats), _ptr(ws), nbytes)
    return loss, stats


def _ds_backward(x: Tensor, teacher: Tensor, index: Tensor, stats: Tensor, g_loss: Tensor, ref) -> Tensor:
    grad = torch.empty_like(x)
    g_loss = g_loss.contiguous()
    _call(x.device, "dw_distill_bwd", ref, x.data_ptr(), teacher.data_ptr(), index.data_ptr(), stats.data_ptr(),
          g_loss.data_ptr(), grad.data_ptr())
    return grad


def _ds_node_backward(ctx, g_loss):
    logits, teacher, index = ctx.saved_tensors
    x = logits if ctx.in_place else logits.contiguous()
    return _ds_backward(x, teacher, index, ctx.stats, g_loss, ctx.ref), None, None, None, None, None


class _DistillFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher, index, dim, scale, renormalise):
        x, teacher, index, (ctx.ref, nbytes) = _ds_desc(logits, teacher, index, dim, scale, renormalise)
        loss, ctx.stats = _ds_forward(x, teacher, index, dim, True, ctx.ref, nbytes)
        ctx.save_for_backward(logits, teacher, index)
        ctx.in_place = x is logits
        return loss

    backward = staticmethod(_once(_ds_node_backward))


@torch.library.custom_op("depthwarp::distill_loss", mutates_args=())
def _distill_op(logits: Tensor, teacher: Tensor, index: Tensor, dim: int, scale: float,
                renormalise: bool) -> Tuple[Tensor, Tensor]:
    x, teacher, index, plan = _ds_desc(logits, teacher, index, dim, scale, renormalise)
    return _ds_forward(x, teacher, index, dim, True, *plan)


@_distill_op.register_fake
def _(logits, teacher, index, dim, scale, renormalise):
    rows = _rows_shape(logits, dim)
    return logits.new_empty(rows, dtype=torch.float32), logits.new_empty(rows + (4,), dtype=torch.float32)


@torch.library.custom_op("depthwarp::distill_loss_bwd", mutates_args=())
def _distill_bwd_op(logits: Tensor, teacher: Tensor, index: Tensor, stats: Tensor, g_loss: Tensor, dim: int,
                    scale: float, renormalise: bool) -> Tensor:
    x, teacher, index, (ref, _) = _ds_desc(logits, teacher, index, dim, scale, renormalise)
    return _ds_backward(x, teacher, index, stats, g_loss, ref)


@_distill_bwd_op.register_fake
def _(logits, teacher, index, stats, g_loss, dim, scale, renormalise):
    return torch.empty_like(_place(logits, dim)[0])


def _ds_setup(ctx, inputs, output):
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(*inputs[:3], output[1])
    ctx.args = inputs[3:]


def _ds_op_backward(ctx, g_loss, _g_stats):
    logits, teacher, index, stats = ctx.saved_tensors
    return _distill_bwd_op(logits, teacher, index, stats, g_loss, *ctx.args), None, None, None, None, None


_distill_op.register_autograd(_ds_op_backward, setup_context=_ds_setup)


def distill_loss(logits: Tensor, teacher: Tensor, teacher_index: Tensor, *, dim: int = 1, scale: float = 1.0,
                 renormalise: bool = False) -> Tensor:
    """Kullback-Leibler divergence of a student from a teacher that is known by its top entries.

    `teacher` (float32, bfloat16 or float16 log-probabilities) and `teacher_index` (int32 or int64 classes)
    have the shape of `logits` with 1 to 64 entries in place of the classes along `dim`; entries with
    an index outside [0, classes) are padding, whatever their value.  Everything the teacher does not
    list is one further class: it has the teacher's remaining probability and the sum of the student's.
    With `renormalise` the teacher's distribution is the soft-max of its listed values (then they may
    be logits, too), and no probability is left for the rest.

    Returns the loss of every row (the shape of `logits` without `dim`, float32), differentiable with
    respect to `logits`, once; the teacher is a constant and must not require a gradient.  A row
    without entries has loss and gradient 0.  A class listed twice counts with both entries.  The loss
    is +inf where the teacher lists a class the student has at -inf.
    """
    dim, scale = _check_logits(logits, dim, scale)
    if teacher.dtype not in _TEACHER_FLAGS:
        raise TypeError(f"teacher: expected float32, bfloat16 or float16, got {teacher.dtype}")
    k = teacher.shape[dim] if teacher.dim() == logits.dim() else 0
    shape = logits.shape[:dim] + (k,) + logits.shape[dim + 1:]
    if not 1 <= k <= _lib.DW_DIST_MAX_ENTRIES or teacher.shape != shape:
        raise ValueError(f"teacher: expected the shape of the logits {tuple(logits.shape)} with 1 to "
                         f"{_lib.DW_DIST_MAX_ENTRIES} entries along axis {dim}, got {tuple(teacher.shape)}")
    if teacher.device != logits.device:
        raise ValueError(f"teacher: expected a tensor on {logits.device}, got {teacher.device}")
    _check_index("teacher_index", teacher_index, teacher.shape, logits.device)
    grad = torch.is_grad_enabled()
    if grad and teacher.requires_grad:
        raise ValueError("teacher: no gradient flows to the teacher; pass teacher.detach()")
    renormalise = bool(renormalise)
    if torch.compiler.is_compiling():
        return _distill_op(logits, teacher, teacher_index, dim, scale, renormalise)[0]
    if grad and logits.requires_grad:
        return _DistillFunction.apply(logits, teacher, teacher_index, dim, scale, renormalise)
    x, teacher, teacher_index, plan = _ds_desc(logits, teacher, teacher_index, dim, scale, renormalise)
    return _ds_forward(x, teacher, teacher_index, dim, False, *plan)[0]
