"""Distributions over classes -- the disparity bins of a volume, or any other soft-max axis -- as HIP
kernels: scoring (log-probability of a given class, entropy, top alternatives) and distillation from
a teacher known by its top entries, both differentiable.

They stand next to the disparity regression of `disparity.soft_argmin` (the reference's
model/model.py:417-429, 454-456; the reference itself has neither operator):

    teacher = log_probs(teacher_cost, scale=-1.0, top=8)                    # 64 bytes a pixel instead of 4 D
    loss = distill_loss(student_cost, teacher.top_log_prob, teacher.top_index, scale=-1.0)   # (B, H, W)
    nll = -log_probs(student_cost, true_bin, scale=-1.0).log_prob           # 0 where true_bin is no bin
    (loss + nll).mean().backward()

Logits are float32, bfloat16 or float16; the class axis is `dim` (1, as in a (B, D, H, W) volume or a
(rows, classes) matrix), and `scale * logits` are the log-weights: -1 for a cost volume, 1/T for a
temperature (of either sign, |scale| from 2^-120 to 2^120).  Tensors in memory order, or with the class
axis last in memory (torch's channels_last), are read where they are; any other order is copied first.
Sums and results are float32, gradients have the type and the order of the logits (memory order, where
those were copied).

A volume in memory order is read by a block for every 64 pixels.  One of few pixels and thousands of classes
leaves most of the chip idle that way: give it with the class axis last in memory (1 x 32768 x 64 bfloat16: 148 us
in memory order, 8 us that way, 11 us for the copy).

Tracers and dispatch modes (torch.compile, make_fx, torch.export, torch.jit.trace, FakeTensorMode) see
registered operators with the same results; eager calls refuse functorch's transforms.

Calls can be captured into a graph, backward passes with them; workspaces belong to the call, so graphs do
not share them.  While a backward pass is captured, no eager graph of the same leaves may be alive (torch
ends the process): drop the eager results first, or capture `torch.autograd.grad`.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import struct
from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor

from . import _lib

__all__ = ["LogProbs", "log_probs", "distill_loss"]

_DTYPES = {torch.float32: _lib.DW_DTYPE_F32, torch.bfloat16: _lib.DW_DTYPE_BF16, torch.float16: _lib.DW_DTYPE_F16}
_TEACHER_FLAGS = {torch.float32: 0, torch.bfloat16: _lib.DW_DIST_TEACHER_BF16, torch.float16: _lib.DW_DIST_TEACHER_F16}
_INDEX_FLAGS = {torch.int32: 0, torch.int64: _lib.DW_DIST_INDEX64}


class LogProbs(NamedTuple):
    log_prob: Optional[Tensor]       # of the given class; 0 where none is given; None without an index
    entropy: Tensor                  # of the row's distribution, in nats
    top_log_prob: Optional[Tensor]   # the `top` most likely classes along the class axis, descending; None for top = 0
    top_index: Optional[Tensor]      # their indices, int32; ties: the lowest first


# Host time counts: a small training step is bound by it.  What a call's shapes and types decide -- every check,
# the descriptor, the workspace's size -- is worked out once and kept by them (`_lp_plan`, `_ds_plan`), and an eager
# call's outputs, launches and autograd node are made in C++ (csrc/distribution_autograd.cpp).

@functools.lru_cache(maxsize=None)
def _eager():
    """The two eager calls of libdepthwarp_torch.so, bound to the library in use."""
    path = _lib.LIB_PATH.parent / "libdepthwarp_torch.so"
    if not path.exists():
        path = _lib._PKG / "libdepthwarp_torch.so"
    if not path.exists():
        raise _lib.DepthwarpError(f"{path} is missing: build it with `python -m depth_estimation_amd.build`. "
                                  "There is no Python fallback for these calls.")
    torch.ops.load_library(str(path))
    lib = _lib.lib()
    torch.ops.depthwarp._bind_distribution(*(C.cast(getattr(lib, n), C.c_void_p).value for n in (
        "dw_strerror", "dw_log_probs_fwd", "dw_log_probs_bwd", "dw_distill_fwd", "dw_distill_bwd")))
    return torch.ops.depthwarp._log_probs_eager.default, torch.ops.depthwarp._distill_eager.default


_PLAIN = (Tensor, torch.nn.Parameter)
_modes, _is_tracing = torch._C._len_torch_dispatch_stack, torch._C._is_tracing


def _watched(a: Tensor, b: Optional[Tensor], c: Optional[Tensor] = None) -> bool:
    """Whether something records or replaces tensor operations (torch.compile, a dispatch mode such as make_fx's or a
    FakeTensorMode, torch.jit.trace, tensors of another class): it has to see the registered operators."""
    return (torch.compiler.is_compiling() or _modes() > 0 or _is_tracing() or type(a) not in _PLAIN
            or (b is not None and type(b) not in _PLAIN) or (c is not None and type(c) not in _PLAIN))


def _call(device: torch.device, fn, *args) -> None:
    """One library call on the device's current stream (the library launches on the current device)."""
    with torch.cuda.device(device):
        rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    _lib.check(rc, fn.__name__)


def _workspace(x: Tensor, nbytes: int) -> Optional[Tensor]:
    # allocated for each call: calls on other streams, or captured into other graphs, have their own
    return torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None


class _Plan(NamedTuple):
    """What shapes and types decide."""
    layout: int        # _IN_PLACE, _LAST, or _COPY: how the kernels read the logits
    dim: int
    rows: tuple        # shape without the class axis
    ref: object        # descriptor, for ctypes
    call: tuple        # for C++: the words of its Call -- descriptor, workspace, class axis, entries, layouts
    nbytes: int        # workspace
    top: int = 0
    list_layout: int = 0      # distillation: the same of the teacher's tensors (_COPY where they have no common order)


def _plan(layout: int, dim: int, shape, descriptor, top: int = 0, list_layout: int = 0) -> _Plan:
    ref, words, nbytes = descriptor
    return _Plan(layout, dim, tuple(shape[:dim]) + tuple(shape[dim + 1:]), ref,
                 words + (nbytes, dim, top, layout, list_layout), nbytes, top, list_layout)


_IN_PLACE, _LAST, _COPY = 0, 1, 2


def _contiguous(shape, stride) -> bool:
    n = 1
    for size, step in zip(reversed(shape), reversed(stride)):
        if size != 1:
            if step != n:
                return 0 in shape
            n *= size
    return True


def _moved(t, dim):
    """Sizes or strides with the class axis moved to the end."""
    return tuple(t[:dim]) + tuple(t[dim + 1:]) + (t[dim],)


def _layout(shape, stride, dim: int) -> int:
    if _contiguous(shape, stride):
        return _IN_PLACE
    return _LAST if _contiguous(_moved(shape, dim), _moved(stride, dim)) else _COPY


def _descriptor(workspace_of: str, shape, dim: int, last: bool, dtype, scale: float, entries: int, flags: int,
                stride=(0, 0, 0)):
    if last:
        flags |= _lib.DW_DIST_LAST
    d = _lib.DwDistDesc(math.prod(shape[:dim]), shape[dim], math.prod(shape[dim + 1:]), stride, scale, _DTYPES[dtype],
                        entries, flags)
    ref = C.byref(d)
    nbytes = getattr(_lib.lib(), workspace_of)(ref)
    if nbytes < 0:
        _lib.check(int(nbytes), f"{workspace_of}(shape={tuple(shape)}, entries={entries}, scale={scale})")
    return ref, struct.unpack(f"{C.sizeof(d) // 8}q", bytes(d)), nbytes


def _check_problem(shape, dtype, dim: int, scale: float) -> int:
    if dtype not in _DTYPES:
        raise TypeError(f"logits: expected float32, bfloat16 or float16, got {dtype}")
    n = len(shape)
    if not -n <= dim < n:
        raise ValueError(f"dim: no axis {dim} in logits of shape {tuple(shape)}")
    dim %= n
    if shape[dim] == 0:
        raise ValueError(f"logits: no classes along axis {dim} of {tuple(shape)}")
    if not math.isfinite(scale) or scale == 0.0:
        raise ValueError(f"scale: expected a finite number other than 0, got {scale}")
    return dim


def _check_index(name: str, dtype, shape, want) -> None:
    if dtype not in _INDEX_FLAGS:
        raise TypeError(f"{name}: expected int32 or int64, got {dtype}")
    if tuple(shape) != tuple(want):
        raise ValueError(f"{name}: expected shape {tuple(want)}, got {tuple(shape)}")


def _check_device(logits: Tensor, **others: Optional[Tensor]) -> None:
    if not logits.is_cuda:
        raise _lib.DepthwarpError(f"logits: expected a ROCm device tensor, got {logits.device} "
                                  "(the HIP kernels have no CPU path)")
    for name, t in others.items():
        if t is not None and t.device != logits.device:
            raise ValueError(f"{name}: expected a tensor on {logits.device}, got {t.device}")


# ------------------------------------------------------------------------------ log-probabilities

def _lp_check(shape, dtype, index_dtype, index_shape, dim: int, scale: float, top: int) -> int:
    dim = _check_problem(shape, dtype, dim, scale)
    most = min(_lib.DW_DIST_MAX_ENTRIES, shape[dim])
    if not 0 <= top <= most:
        raise ValueError(f"top: expected 0 to {most}, got {top}")
    if index_dtype is not None:
        _check_index("index", index_dtype, index_shape, tuple(shape[:dim]) + tuple(shape[dim + 1:]))
    return dim


def _make_lp_plan(shape, stride, dtype, index_dtype, index_shape, dim: int, scale: float, top: int) -> _Plan:
    dim = _lp_check(shape, dtype, index_dtype, index_shape, dim, scale, top)
    layout = _layout(shape, stride, dim)
    flags = 0 if index_dtype is None else _INDEX_FLAGS[index_dtype]
    return _plan(layout, dim, shape, _descriptor("dw_log_probs_workspace_bytes", shape, dim, layout == _LAST, dtype, scale, top,
                                                 flags), top)


_lp_plan = functools.lru_cache(maxsize=512)(_make_lp_plan)


def _plan_of(logits: Tensor, index: Optional[Tensor], dim: int, scale: float, top: int) -> _Plan:
    if index is None:
        return _lp_plan(logits.shape, logits.stride(), logits.dtype, None, None, dim, scale, top)
    return _lp_plan(logits.shape, logits.stride(), logits.dtype, index.dtype, index.shape, dim, scale, top)


def _lp_forward(logits: Tensor, index: Optional[Tensor], plan: _Plan):
    x = logits.contiguous() if plan.layout == _COPY else logits
    dev, rows, top = x.device, plan.rows, plan.top
    ent = torch.empty(rows, dtype=torch.float32, device=dev)
    stats = torch.empty(rows + (3,), dtype=torch.float32, device=dev)
    lp = lp_ptr = index_ptr = top_lp = top_lp_ptr = top_idx = top_idx_ptr = None
    if index is not None:
        index = index.contiguous()
        index_ptr = index.data_ptr()
        lp = torch.empty(rows, dtype=torch.float32, device=dev)
        lp_ptr = lp.data_ptr()
    if top:
        if plan.layout == _LAST:   # the kernels write the list of a row together, too
            top_lp = torch.empty(rows + (top,), dtype=torch.float32, device=dev).movedim(-1, plan.dim)
            top_idx = torch.empty(rows + (top,), dtype=torch.int32, device=dev).movedim(-1, plan.dim)
        else:
            shape = rows[:plan.dim] + (top,) + rows[plan.dim:]
            top_lp = torch.empty(shape, dtype=torch.float32, device=dev)
            top_idx = torch.empty(shape, dtype=torch.int32, device=dev)
        top_lp_ptr, top_idx_ptr = top_lp.data_ptr(), top_idx.data_ptr()
    ws = _workspace(x, plan.nbytes)
    _call(dev, _lib.lib().dw_log_probs_fwd, plan.ref, x.data_ptr(), index_ptr, lp_ptr, ent.data_ptr(), top_lp_ptr,
          top_idx_ptr, stats.data_ptr(), None if ws is None else ws.data_ptr(), plan.nbytes)
    return lp, ent, top_lp, top_idx, stats


def _lp_backward(logits: Tensor, index: Optional[Tensor], stats: Tensor, g_lp: Optional[Tensor],
                 g_ent: Optional[Tensor], plan: _Plan) -> Tensor:
    x = logits.contiguous() if plan.layout == _COPY else logits
    grad, stats = torch.empty_like(x), stats.contiguous()
    index_ptr = g_lp_ptr = g_ent_ptr = None
    if index is not None:
        index = index.contiguous()
        index_ptr = index.data_ptr()
        if g_lp is not None:
            g_lp = g_lp.contiguous()
            g_lp_ptr = g_lp.data_ptr()
    if g_ent is not None:
        g_ent = g_ent.contiguous()
        g_ent_ptr = g_ent.data_ptr()
    _call(x.device, _lib.lib().dw_log_probs_bwd, plan.ref, x.data_ptr(), index_ptr, stats.data_ptr(), g_lp_ptr,
          g_ent_ptr, grad.data_ptr())
    return grad


# Torch operators with the same results, which is what tracers record.  An operator always returns tensors:
# without an index, log_prob is empty; the last result is for the backward pass.

@torch.library.custom_op("depthwarp::log_probs", mutates_args=())
def _log_probs_op(logits: Tensor, index: Optional[Tensor], dim: int, scale: float,
                  top: int) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    lp, ent, top_lp, top_idx, stats = _lp_forward(logits, index, _plan_of(logits, index, dim, scale, top))
    if lp is None:
        lp = ent.new_empty((0,))
    if not top:
        top_lp, top_idx = ent.new_empty((0,)), ent.new_empty((0,), dtype=torch.int32)
    return lp, ent, top_lp, top_idx, stats


@_log_probs_op.register_fake
def _(logits, index, dim, scale, top):
    dim %= logits.dim()
    rows = logits.shape[:dim] + logits.shape[dim + 1:]
    ent = logits.new_empty(rows, dtype=torch.float32)
    lp = torch.empty_like(ent) if index is not None else ent.new_empty((0,))
    if not top:
        top_lp, top_idx = ent.new_empty((0,)), ent.new_empty((0,), dtype=torch.int32)
    elif not logits.is_contiguous() and logits.movedim(dim, -1).is_contiguous():
        top_lp = ent.new_empty(rows + (top,)).movedim(-1, dim)
        top_idx = ent.new_empty(rows + (top,), dtype=torch.int32).movedim(-1, dim)
    else:
        shape = logits.shape[:dim] + (top,) + logits.shape[dim + 1:]
        top_lp, top_idx = ent.new_empty(shape), ent.new_empty(shape, dtype=torch.int32)
    return lp, ent, top_lp, top_idx, ent.new_empty(rows + (3,))


def _fake_grad(logits: Tensor, dim: int) -> Tensor:
    in_place = logits.is_contiguous() or logits.movedim(dim, -1).is_contiguous()
    return torch.empty_like(logits) if in_place else torch.empty_like(logits, memory_format=torch.contiguous_format)


@torch.library.custom_op("depthwarp::log_probs_bwd", mutates_args=())
def _log_probs_bwd_op(logits: Tensor, index: Optional[Tensor], stats: Tensor, g_lp: Optional[Tensor],
                      g_ent: Optional[Tensor], dim: int, scale: float) -> Tensor:
    return _lp_backward(logits, index, stats, g_lp, g_ent, _plan_of(logits, index, dim, scale, 0))


@_log_probs_bwd_op.register_fake
def _(logits, index, stats, g_lp, g_ent, dim, scale):
    return _fake_grad(logits, dim)


def _lp_setup(ctx, inputs, output):
    logits, index, dim, scale, _top = inputs
    ctx.mark_non_differentiable(*output[2:])
    ctx.save_for_backward(logits, index, output[4])
    ctx.dim, ctx.scale = dim, scale


def _lp_op_backward(ctx, g_lp, g_ent, _g_top, _g_index, _g_stats):
    logits, index, stats = ctx.saved_tensors
    return _log_probs_bwd_op(logits, index, stats, g_lp, g_ent, ctx.dim, ctx.scale), None, None, None, None


_log_probs_op.register_autograd(_lp_op_backward, setup_context=_lp_setup)


def log_probs(logits: Tensor, index: Optional[Tensor] = None, *, dim: int = 1, scale: float = 1.0,
              top: int = 0) -> LogProbs:
    """Scores rows of `logits` against the classes `index` and describes their distribution.

    `index` (int32 or int64) has the shape of `logits` without `dim`; a value outside [0, classes) means
    that no class is given there (a pixel without ground truth, or beyond the range): log-probability 0 and
    no gradient.  The `top` (0 to 64) most likely classes come back as log-probabilities and int32 indices, in
    descending order, equal values by lowest index.

    `log_prob` and `entropy` are differentiable with respect to `logits`, once; the top lists are not.
    A class at -inf has probability 0; a row of nothing else has entropy 0, log-probability -inf and
    gradient 0.  A row with NaN (or +inf) has NaN results.  A row that gets no upstream gradient gets
    zeros whatever it holds.
    """
    if not logits.is_cuda or (index is not None and index.device != logits.device):
        _check_device(logits, index=index)
    scale, top = float(scale), int(top)
    if _watched(logits, index):
        dim = _lp_check(logits.shape, logits.dtype, None if index is None else index.dtype,
                        None if index is None else index.shape, dim, scale, top)
        lp, ent, top_lp, top_idx, _ = _log_probs_op(logits, index, dim, scale, top)
        return LogProbs(None if index is None else lp, ent, top_lp if top else None, top_idx if top else None)
    plan = _plan_of(logits, index, dim, scale, top)
    out = _eager()[0](logits, index, plan.call, plan.rows)
    if index is None:
        return LogProbs(None, *out) if top else LogProbs(None, out[0], None, None)
    return LogProbs(*out) if top else LogProbs(*out, None, None)


# --------------------------------------------------------------------------------- distillation

def _ds_check(shape, dtype, t_shape, t_dtype, i_shape, i_dtype, dim: int, scale: float) -> int:
    dim = _check_problem(shape, dtype, dim, scale)
    if t_dtype not in _TEACHER_FLAGS:
        raise TypeError(f"teacher: expected float32, bfloat16 or float16, got {t_dtype}")
    k = t_shape[dim] if len(t_shape) == len(shape) else 0
    want = tuple(shape[:dim]) + (k,) + tuple(shape[dim + 1:])
    if not 1 <= k <= _lib.DW_DIST_MAX_ENTRIES or tuple(t_shape) != want:
        raise ValueError(f"teacher: expected the shape of the logits {tuple(shape)} with 1 to "
                         f"{_lib.DW_DIST_MAX_ENTRIES} entries along axis {dim}, got {tuple(t_shape)}")
    _check_index("teacher_index", i_dtype, i_shape, want)
    return dim


def _make_ds_plan(shape, stride, dtype, t_shape, t_stride, t_dtype, i_shape, i_stride, i_dtype, dim: int,
                  scale: float, renormalise: bool) -> _Plan:
    dim = _ds_check(shape, dtype, t_shape, t_dtype, i_shape, i_dtype, dim, scale)
    k, inner = t_shape[dim], math.prod(t_shape[dim + 1:])
    # the list's element strides along outer, entry, inner: its tensors as they are if they share an order
    t_layout, i_layout = _layout(t_shape, t_stride, dim), _layout(i_shape, i_stride, dim)
    list_layout = t_layout if t_layout == i_layout else _COPY
    strides = (k * inner, 1, k) if list_layout == _LAST else (k * inner, inner, 1)
    layout = _layout(shape, stride, dim)
    flags = _INDEX_FLAGS[i_dtype] | _TEACHER_FLAGS[t_dtype] | (_lib.DW_DIST_RENORMALISE if renormalise else 0)
    return _plan(layout, dim, shape, _descriptor("dw_distill_workspace_bytes", shape, dim, layout == _LAST, dtype, scale, k,
                                                 flags, strides), list_layout=list_layout)


_ds_plan = functools.lru_cache(maxsize=512)(_make_ds_plan)


def _ds_plan_of(logits: Tensor, teacher: Tensor, index: Tensor, dim: int, scale: float, renormalise: bool) -> _Plan:
    return _ds_plan(logits.shape, logits.stride(), logits.dtype, teacher.shape, teacher.stride(), teacher.dtype,
                    index.shape, index.stride(), index.dtype, dim, scale, renormalise)


def _ds_forward(logits: Tensor, teacher: Tensor, index: Tensor, plan: _Plan):
    x = logits.contiguous() if plan.layout == _COPY else logits
    if plan.list_layout == _COPY:
        teacher, index = teacher.contiguous(), index.contiguous()
    loss = torch.empty(plan.rows, dtype=torch.float32, device=x.device)
    stats = torch.empty(plan.rows + (4,), dtype=torch.float32, device=x.device)
    ws = _workspace(x, plan.nbytes)
    _call(x.device, _lib.lib().dw_distill_fwd, plan.ref, x.data_ptr(), teacher.data_ptr(), index.data_ptr(),
          loss.data_ptr(), stats.data_ptr(), None if ws is None else ws.data_ptr(), plan.nbytes)
    return loss, stats


def _ds_backward(logits: Tensor, teacher: Tensor, index: Tensor, stats: Tensor, g_loss: Tensor, plan: _Plan) -> Tensor:
    x = logits.contiguous() if plan.layout == _COPY else logits
    if plan.list_layout == _COPY:
        teacher, index = teacher.contiguous(), index.contiguous()
    grad = torch.empty_like(x)
    stats, g_loss = stats.contiguous(), g_loss.contiguous()
    _call(x.device, _lib.lib().dw_distill_bwd, plan.ref, x.data_ptr(), teacher.data_ptr(), index.data_ptr(),
          stats.data_ptr(), g_loss.data_ptr(), grad.data_ptr())
    return grad


@torch.library.custom_op("depthwarp::distill_loss", mutates_args=())
def _distill_op(logits: Tensor, teacher: Tensor, index: Tensor, dim: int, scale: float,
                renormalise: bool) -> Tuple[Tensor, Tensor]:
    return _ds_forward(logits, teacher, index, _ds_plan_of(logits, teacher, index, dim, scale, renormalise))


@_distill_op.register_fake
def _(logits, teacher, index, dim, scale, renormalise):
    dim %= logits.dim()
    rows = logits.shape[:dim] + logits.shape[dim + 1:]
    return logits.new_empty(rows, dtype=torch.float32), logits.new_empty(rows + (4,), dtype=torch.float32)


@torch.library.custom_op("depthwarp::distill_loss_bwd", mutates_args=())
def _distill_bwd_op(logits: Tensor, teacher: Tensor, index: Tensor, stats: Tensor, g_loss: Tensor, dim: int,
                    scale: float, renormalise: bool) -> Tensor:
    return _ds_backward(logits, teacher, index, stats, g_loss,
                        _ds_plan_of(logits, teacher, index, dim, scale, renormalise))


@_distill_bwd_op.register_fake
def _(logits, teacher, index, stats, g_loss, dim, scale, renormalise):
    return _fake_grad(logits, dim)


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
    is +inf where the teacher gives a listed class probability and the student has it at -inf.  The rest is
    different: where the student has no possible class outside the list, the teacher's remaining
    probability adds nothing to the loss and to the gradient, as if there were no further class.
    """
    if not (logits.is_cuda and teacher.device == logits.device == teacher_index.device):
        _check_device(logits, teacher=teacher, teacher_index=teacher_index)
    scale, renormalise = float(scale), bool(renormalise)
    if teacher.requires_grad and torch.is_grad_enabled():
        raise ValueError("teacher: no gradient flows to the teacher; pass teacher.detach()")
    if _watched(logits, teacher, teacher_index):
        dim = _ds_check(logits.shape, logits.dtype, teacher.shape, teacher.dtype, teacher_index.shape,
                        teacher_index.dtype, dim, scale)
        return _distill_op(logits, teacher, teacher_index, dim, scale, renormalise)[0]
    plan = _ds_plan_of(logits, teacher, teacher_index, dim, scale, renormalise)
    return _eager()[1](logits, teacher, teacher_index, plan.call, plan.rows)
