"""Training operators on the B200 kernels: layer norm, adaptive layer norm, gradient clipping.

The planner plans with a world model that its user trains and fine-tunes in torch. These are the
memory-bound operators of that step around its matrix products:

* ``layer_norm`` -- ``nn.LayerNorm`` over the last dim, with the gradients of input, weight and bias
  (reference ``lewm/module.py:44,79,147``).
* ``ada_layer_norm`` -- ``modulate(norm(x), shift, scale)`` of the AdaLN-conditioned predictor block
  (reference ``lewm/module.py:6-8,96-110``), with the gradients of input, shift and scale.
* ``grad_norm`` / ``clip_grads`` / ``clip_grad_norm_`` -- the global norm of many gradients taken as
  one vector, and scaling by it.
* ``install_training_norms(model)`` -- routes the LayerNorms and conditional blocks of a torch world
  model (a reference ``JEPA``) through the first two, forward and backward.

Tensors are float32, bfloat16 or float16 CUDA tensors; arithmetic, statistics and sums are float32
(the norm's sum float64) and every result is rounded once. Calls run on the current stream of
their tensors' device, allocate from torch's caching allocator, never synchronize (except
``error_if_nonfinite``) and can be captured into CUDA graphs. Results do not depend on the run:
no atomics. As with torch's own operators, a caller that hands tensors to another stream orders
the streams. There is no CPU fallback: CPU tensors raise ``ValueError``.
"""

from __future__ import annotations

import ctypes as C
import functools
import math
from typing import Any, Iterable, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _lib

TYPE_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # LEWM_TYPE_*
NORM_KIND = {2.0: 0, math.inf: 1}  # LEWM_NORM_L2, LEWM_NORM_MAX


def _check_tensor(name: str, t: torch.Tensor, device: Optional[torch.device] = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype not in TYPE_CODE:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.layout is not torch.strided:
        raise ValueError(f"{name} must be a dense tensor, got layout {t.layout}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, x on {device}")


def _need_cuda(t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise ValueError(f"the B200 training operators need a CUDA device, got {t.device}")


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """``t`` as rows of its last dim and the elements between them, copied only where the leading
    dims do not step evenly through memory or the last dim is not dense."""
    if t.is_contiguous():
        return t, t.shape[-1]
    if t.stride(-1) == 1 or t.shape[-1] == 1:
        step, extent = None, 1  # stride of the rows so far, and how many there are
        for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if step is None:
                step = stride
            elif stride != step * extent:
                break
            extent *= size
        else:
            return t, t.shape[-1] if step is None else step
    return t.contiguous(), t.shape[-1]


def _call_forward(x: torch.Tensor, a, b, eps: float, group: int, stats: Optional[torch.Tensor]) -> torch.Tensor:
    width = x.shape[-1]
    rows = x.numel() // width
    x, xs = _rows(x)
    as_ = bs = 0
    p_type = 0
    for p in (a, b):
        if p is not None:
            p_type = TYPE_CODE[p.dtype]
    if a is not None:
        a, as_ = _rows(a)
    if b is not None:
        b, bs = _rows(b)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if rows:
        desc = _lib.NormDescC(rows, width, xs, group, as_, bs, TYPE_CODE[x.dtype], p_type, eps)
        device = x.device
        _lib.check(_lib.lib().lewm_norm_forward(
            C.byref(desc), x.data_ptr(), None if a is None else a.data_ptr(), None if b is None else b.data_ptr(),
            y.data_ptr(), None if stats is None else stats.data_ptr(), device.index,
            torch.cuda.current_stream(device).cuda_stream))
    return y


class _Norm(torch.autograd.Function):
    """y = z a + b (``group`` 0) or z (1 + a) + b, a row of a and b for ``group`` rows of x."""

    @staticmethod
    def forward(ctx, x, a, b, eps, group):
        width = x.shape[-1]
        x = _rows(x)[0].detach()  # the copy, where one is needed, serves the backward pass too
        stats = torch.empty(2, x.numel() // width, dtype=torch.float32, device=x.device)
        y = _call_forward(x, a, b, eps, group, stats)
        ctx.save_for_backward(x, a, stats)
        ctx.meta = (eps, group, None if b is None else b.shape, None if b is None else b.dtype)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, a, stats = ctx.saved_tensors
        eps, group, b_shape, b_dtype = ctx.meta
        need_x, need_a, need_b = ctx.needs_input_grad[:3]
        device, width = x.device, x.shape[-1]
        rows = x.numel() // width
        dx = torch.empty(x.shape, dtype=x.dtype, device=device) if need_x else None
        da = torch.empty(a.shape, dtype=a.dtype, device=device) if need_a else None
        db = db_out = None
        if need_b:
            if group == 1 and b_dtype is dy.dtype and rows:
                db = dy.reshape(b_shape)  # a shift row per row of x: its gradient is dy
            else:
                db = db_out = torch.empty(b_shape, dtype=b_dtype, device=device)
        if rows == 0:
            for g in (da, db_out):
                if g is not None:
                    g.zero_()
        elif dx is not None or da is not None or db_out is not None:
            dy, ds = _rows(dy)
            x, xs = _rows(x)
            as_ = 0
            p_type = 0 if b_dtype is None else TYPE_CODE[b_dtype]
            if a is not None:
                a, as_ = _rows(a)
                p_type = TYPE_CODE[a.dtype]
            desc = _lib.NormDescC(rows, width, xs, group, as_, 0, TYPE_CODE[x.dtype], p_type, eps)
            ref = C.byref(desc)
            lib = _lib.lib()
            ws, size = None, 0
            if da is not None or db_out is not None:
                size = lib.lewm_norm_workspace(ref)
                if size:
                    ws = torch.empty(size, dtype=torch.uint8, device=device)
            _lib.check(lib.lewm_norm_backward(
                ref, dy.data_ptr(), ds, x.data_ptr(), None if a is None else a.data_ptr(), stats.data_ptr(),
                None if dx is None else dx.data_ptr(), None if da is None else da.data_ptr(),
                None if db_out is None else db_out.data_ptr(), None if ws is None else ws.data_ptr(), size,
                device.index, torch.cuda.current_stream(device).cuda_stream))
        return dx, da, db, None, None


def _norm(x, a, b, eps: float, group: int) -> torch.Tensor:
    _need_cuda(x)
    if torch.is_grad_enabled() and (x.requires_grad or (a is not None and a.requires_grad)
                                    or (b is not None and b.requires_grad)):
        return _Norm.apply(x, a, b, eps, group)
    return _call_forward(x, a, b, eps, group, None)


def _check_eps(eps: float) -> float:
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must be finite and >= 0, got {eps}")
    return eps


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``nn.LayerNorm`` over the last dim of ``x``: ``(x - mean) / sqrt(var + eps) * weight + bias``.

    ``weight`` and ``bias`` are (D,) of one type, float32 or any other, each optional. The result has
    the shape and type of ``x`` and is contiguous. ``x`` may be strided: rows that step evenly
    through memory are read in place, others are copied first. Differentiable once in all three.
    """
    _check_tensor("x", x)
    if x.ndim == 0 or x.shape[-1] == 0:
        raise ValueError(f"x must have a last dim of at least 1, got shape {tuple(x.shape)}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        _check_tensor(name, p, x.device)
        if tuple(p.shape) != (x.shape[-1],):
            raise ValueError(f"{name} must be ({x.shape[-1]},), got {tuple(p.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    weight = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    bias = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    return _norm(x, weight, bias, _check_eps(eps), 0)


def ada_layer_norm(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``modulate(norm(x), shift, scale)``: ``(x - mean) / sqrt(var + eps) * (1 + scale) + shift``.

    ``shift`` and ``scale`` have one shape and type (float32 or any other): that of ``x``, or with
    size 1 in any number of dims right before the last, so that a modulation row serves the rows of
    ``x`` under it ((B, 1, D) for x (B, T, D); (D,) for all rows). Leading dims of size 1 may be
    left out. Chunks of an AdaLN Linear's output are read in place. The result has the shape and
    type of ``x`` and is contiguous; differentiable once in all three.
    """
    _check_tensor("x", x)
    if x.ndim == 0 or x.shape[-1] == 0:
        raise ValueError(f"x must have a last dim of at least 1, got shape {tuple(x.shape)}")
    _check_tensor("shift", shift, x.device)
    _check_tensor("scale", scale, x.device)
    if shift.shape != scale.shape or shift.dtype != scale.dtype:
        raise ValueError(f"shift and scale must have one shape and type, got {tuple(shift.shape)} {shift.dtype} and "
                         f"{tuple(scale.shape)} {scale.dtype}")
    group = 1
    if shift.shape != x.shape:
        m = (1,) * (x.ndim - shift.ndim) + tuple(shift.shape)
        shared = len(m) == x.ndim and m[-1] == x.shape[-1]
        i = x.ndim - 2
        while shared and i >= 0 and m[i] == 1:
            group *= x.shape[i]
            i -= 1
        if not shared or m[:i + 1] != tuple(x.shape[:i + 1]):
            raise ValueError(f"shift and scale of shape {tuple(shift.shape)} do not modulate x of shape "
                             f"{tuple(x.shape)}: give a row per row of x, or size 1 in the dims before the last")
    if x.numel() == 0:
        group = 1  # no rows
    return _norm(x, scale, shift, _check_eps(eps), group)


# ---------------------------------------------------------------------------- gradient norm
def _kind(norm_type: float) -> int:
    kind = NORM_KIND.get(float(norm_type))
    if kind is None:
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    return kind


def _check_list(name: str, tensors: Sequence[torch.Tensor]) -> torch.device:
    device = tensors[0].device if isinstance(tensors[0], torch.Tensor) else None
    for i, t in enumerate(tensors):
        if not (isinstance(t, torch.Tensor) and t.dtype in TYPE_CODE and t.device == device
                and t.layout is torch.strided):
            _check_tensor(f"{name}[{i}]", t)
            raise ValueError(f"{name}[{i}] is on {t.device}, {name}[0] on {device}: one device per call")
    return device


def _table(tensors: Sequence[torch.Tensor]):
    """Pointers, element counts and type codes of dense tensors as HOST arrays."""
    n = len(tensors)
    ptr = np.fromiter([t.data_ptr() for t in tensors], np.uint64, n)
    count = np.fromiter([t.numel() for t in tensors], np.int64, n)
    kind = np.fromiter([TYPE_CODE[t.dtype] for t in tensors], np.int32, n)
    return ptr, count, kind


def _overlap(src: np.ndarray, dst: np.ndarray, size: np.ndarray) -> bool:
    """Whether any destination [dst, dst + size) meets another destination or another tensor's source."""
    live = size > 0
    src, dst, size = src[live].astype(np.int64), dst[live].astype(np.int64), size[live]
    order = np.argsort(dst, kind="stable")
    lo, hi = dst[order], dst[order] + size[order]
    if np.any(hi[:-1] > lo[1:]):
        return True
    # Destinations are disjoint and sorted: those a source meets are a range; only its own
    # destination, lying exactly on it, may be in there.
    first = np.searchsorted(hi, src, side="right")
    last = np.searchsorted(lo, src + size, side="left")
    return bool(np.any(last - first != (src == dst)))


def _clip(src, dst, max_norm: float, kind: int, norm_in: Optional[torch.Tensor], device) -> torch.Tensor:
    """The kernels' call: norm of dense ``src``, and with ``dst`` their scaled copies."""
    sp, count, types = _table(src)
    dp = sp if dst is None or dst is src else np.fromiter([t.data_ptr() for t in dst], np.uint64, len(dst))
    if dst is not None and _overlap(sp, dp, count * np.where(types == 0, 4, 2)):
        raise ValueError("gradients overlap in memory (the same one listed twice?), or an output overlaps one")
    _need_cuda(src[0])
    norm = torch.empty((), dtype=torch.float32, device=device)
    ws = torch.empty(_lib.GRAD_WORKSPACE, dtype=torch.uint8, device=device)
    stream = torch.cuda.current_stream(device).cuda_stream
    lib = _lib.lib()
    if dst is None:
        _lib.check(lib.lewm_grad_norm(sp.ctypes.data, count.ctypes.data, types.ctypes.data, len(src), kind,
                                      ws.data_ptr(), norm.data_ptr(), device.index, stream))
        return norm
    _lib.check(lib.lewm_grad_clip(sp.ctypes.data, dp.ctypes.data, count.ctypes.data, types.ctypes.data, len(src), kind,
                                  max_norm, None if norm_in is None else norm_in.data_ptr(), ws.data_ptr(),
                                  norm.data_ptr(), device.index, stream))
    return norm


def _check_max_norm(max_norm: float) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    return max_norm


def grad_norm(grads: Iterable[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all elements of ``grads`` taken as one vector: a 0-d float32 tensor on their device
    (0 on the CPU for no tensors). ``norm_type`` 2 or inf; NaN and infinity propagate."""
    grads = list(grads)
    kind = _kind(norm_type)
    if not grads:
        return torch.tensor(0.0)
    device = _check_list("grads", grads)
    return _clip([t if t.is_contiguous() else t.contiguous() for t in grads], None, 0.0, kind, None, device)


def clip_grads(grads: Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
               out: Optional[Sequence[torch.Tensor]] = None) -> Tuple[List[torch.Tensor], torch.Tensor]:
    """``grads`` scaled by ``min(1, max_norm / (norm + 1e-6))`` and their norm.

    Writes to ``out`` (contiguous tensors of the same shapes and types, which overlap neither each
    other nor ``grads``; or the tensors of ``grads`` themselves) or to new tensors, and returns them.
    """
    grads = list(grads)
    kind = _kind(norm_type)
    max_norm = _check_max_norm(max_norm)
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError(f"out has {len(out)} tensors, grads {len(grads)}")
    if not grads:
        return [], torch.tensor(0.0)
    device = _check_list("grads", grads)
    if out is None:
        out = [torch.empty_like(t, memory_format=torch.contiguous_format, requires_grad=False) for t in grads]
    else:
        for i, (o, g) in enumerate(zip(out, grads)):
            if o is g:
                if not o.is_contiguous():
                    raise ValueError(f"out[{i}] must be contiguous")
                continue
            if not isinstance(o, torch.Tensor) or o.shape != g.shape or o.dtype != g.dtype or o.device != device:
                raise ValueError(f"out[{i}] must be a {g.dtype} tensor of shape {tuple(g.shape)} on {device}")
            if not o.is_contiguous():
                raise ValueError(f"out[{i}] must be contiguous")
    src = [t if t.is_contiguous() else t.contiguous() for t in grads]
    norm = _clip(src, out, max_norm, kind, None, device)
    torch.autograd.graph.increment_version(out)
    return out, norm


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` on the kernels: scales the ``grad`` of every parameter in
    place by ``min(1, max_norm / (norm + 1e-6))`` and returns the norm (0-d float32).

    The gradients are on one CUDA device and do not overlap. ``error_if_nonfinite`` reads the norm
    on the host (so not under graph capture) and raises before anything is scaled."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    kind = _kind(norm_type)
    max_norm = _check_max_norm(max_norm)
    if not grads:
        return torch.tensor(0.0)
    device = _check_list("grad", grads)
    dense = []
    strided = []
    for g in grads:
        if g.is_contiguous():
            dense.append(g)
            continue
        if any(s == 0 and n > 1 for s, n in zip(g.stride(), g.shape)):
            raise ValueError(f"a gradient of shape {tuple(g.shape)} shares memory between its own elements")
        dense.append(g.contiguous())
        strided.append((g, dense[-1]))
    if strided and len({(g.data_ptr(), g.shape, g.stride()) for g in grads}) != len(grads):
        raise ValueError("gradients overlap in memory (the same one listed twice?)")
    norm_in = None
    if error_if_nonfinite:
        norm_in = _clip(dense, None, 0.0, kind, None, device)
        if not math.isfinite(norm_in.item()):
            raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients is non-finite, so it cannot "
                               "be clipped")
    norm = _clip(dense, dense, max_norm, kind, norm_in, device)
    torch.autograd.graph.increment_version(grads)
    with torch.no_grad():
        for g, d in strided:
            g.copy_(d)
    return norm


# ---------------------------------------------------------------------------- a torch world model
def _float32_under_autocast(x: torch.Tensor) -> torch.Tensor:
    """torch runs layer_norm in float32 under autocast."""
    return x.float() if torch.is_autocast_enabled("cuda") and x.dtype in TYPE_CODE else x


def _layer_norm_forward(module: torch.nn.LayerNorm, x: torch.Tensor) -> torch.Tensor:
    return layer_norm(_float32_under_autocast(x), module.weight, module.bias, module.eps)


def _conditional_block_forward(block: torch.nn.Module, x: torch.Tensor, c: torch.Tensor) -> torch.Tensor:
    """``ConditionalBlock.forward`` (reference ``lewm/module.py:105-111``)."""
    shift_a, scale_a, gate_a, shift_m, scale_m, gate_m = block.adaLN_modulation(c).chunk(6, dim=-1)
    x = x + gate_a * block.attn(ada_layer_norm(_float32_under_autocast(x), shift_a, scale_a, block.norm1.eps))
    return x + gate_m * block.mlp(ada_layer_norm(_float32_under_autocast(x), shift_m, scale_m, block.norm2.eps))


def _plain_norm(m: Any) -> bool:
    """A LayerNorm over the last dim without an affine."""
    return isinstance(m, torch.nn.LayerNorm) and len(m.normalized_shape) == 1 and m.weight is None and m.bias is None


class B200TrainingNorms:
    """What ``install_training_norms`` routed: ``modules`` (names), and ``remove()`` to undo it."""

    def __init__(self, model: torch.nn.Module):
        self.modules: List[str] = []
        self._routed: List[torch.nn.Module] = []
        for name, m in model.named_modules():
            if "forward" in m.__dict__:  # routed already, by this or another install
                continue
            if isinstance(m, torch.nn.LayerNorm) and len(m.normalized_shape) == 1:
                m.forward = functools.partial(_layer_norm_forward, m)
            elif (all(hasattr(m, n) for n in ("adaLN_modulation", "attn", "mlp"))
                  and _plain_norm(getattr(m, "norm1", None)) and _plain_norm(getattr(m, "norm2", None))):
                m.forward = functools.partial(_conditional_block_forward, m)
            else:
                continue
            self.modules.append(name)
            self._routed.append(m)

    def remove(self) -> None:
        for m in self._routed:
            m.__dict__.pop("forward", None)
        self._routed = []
        self.modules = []


def install_training_norms(model: torch.nn.Module) -> B200TrainingNorms:
    """Route every ``nn.LayerNorm`` over the last dim and every AdaLN conditional block of ``model``
    (reference ``lewm/module.py:38-53,56-111,131-187,217-240``: predictor, projector heads, and the ViT
    encoder) through ``layer_norm`` and ``ada_layer_norm``, so that a training step of the world
    model runs their forward and backward passes on the B200 kernels. Parameters, state dict and
    autocast behaviour stay as they are: under autocast the norms run in float32 as torch's do.
    The model's inputs must be on a CUDA device."""
    return B200TrainingNorms(model)
