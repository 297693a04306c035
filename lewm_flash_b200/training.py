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
(the gradient norm's sum is float64 over sums of 4 or 8 squares in float32) and every result is rounded
once. Calls run on the current stream of their tensors' device, allocate from torch's caching allocator,
never synchronize (except ``error_if_nonfinite``) and can be captured into CUDA graphs. Results do not
depend on the run: no atomics. As with torch's own operators, a caller that hands tensors to another
stream orders the streams. There is no CPU fallback: CPU tensors raise ``ValueError``.

The norms are differentiable once, in reverse. What would need more raises ``NotImplementedError``
instead of going wrong: forward-mode derivatives, tracers (``torch.jit.trace``, ``make_fx``,
``torch.export``), the transforms of ``torch.func`` and subclasses with a ``__torch_dispatch__``. Other
subclasses and modes see the norms through ``__torch_function__``.
"""

from __future__ import annotations

import dis
import functools
import importlib
import inspect
import types
from typing import Any, Iterable, List, Optional, Sequence, Tuple, Union

import torch
from torch.overrides import handle_torch_function, has_torch_function_variadic

from . import _lib

_ext = None


def _ops():
    """The extension module built from ``csrc/torch_ops.cpp``. Raises if it is missing: there is no
    other implementation to fall back to."""
    global _ext
    if _ext is None:
        _lib.lib()
        try:
            ext = importlib.import_module("lewm_flash_b200._torch_ops")
        except ImportError as e:
            raise RuntimeError("lewm_flash_b200/_torch_ops.so is missing or does not load; build it with "
                               "`python -m lewm_flash_b200.build`") from e
        if ext.abi_version != _lib.ABI_VERSION:
            raise RuntimeError(f"_torch_ops.so was built for C ABI version {ext.abi_version}, this package needs "
                               f"{_lib.ABI_VERSION}; rebuild it")
        _ext = ext
    return _ext


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``nn.LayerNorm`` over the last dim of ``x``: ``(x - mean) / sqrt(var + eps) * weight + bias``.

    ``weight`` and ``bias`` are (D,) of one type, float32 or any other, each optional. The result has
    the shape and type of ``x`` and is contiguous. ``x`` may be strided: rows that step evenly
    through memory are read in place, others are copied first. Differentiable once in all three.
    """
    if has_torch_function_variadic(x, weight, bias):  # subclasses and modes see the call
        return handle_torch_function(layer_norm, (x, weight, bias), x, weight, bias, eps)
    return _ops().layer_norm(x, weight, bias, eps)


def ada_layer_norm(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``modulate(norm(x), shift, scale)``: ``(x - mean) / sqrt(var + eps) * (1 + scale) + shift``.

    ``shift`` and ``scale`` have one shape and type (float32 or any other): that of ``x``, or with
    size 1 in any number of dims right before the last, so that a modulation row serves the rows of
    ``x`` under it ((B, 1, D) for x (B, T, D); (D,) for all rows). Leading dims of size 1 may be
    left out. Chunks of an AdaLN Linear's output are read in place. The result has the shape and
    type of ``x`` and is contiguous; differentiable once in all three.
    """
    if has_torch_function_variadic(x, shift, scale):
        return handle_torch_function(ada_layer_norm, (x, shift, scale), x, shift, scale, eps)
    return _ops().ada_layer_norm(x, shift, scale, eps)


def grad_norm(grads: Iterable[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all elements of ``grads`` taken as one vector: a 0-d float32 tensor on their device
    (0 on the CPU for no tensors). ``norm_type`` 2 or inf; NaN and infinity propagate. Tensors that
    are not contiguous are copied first."""
    return _ops().grad_norm(list(grads), norm_type)


def clip_grads(grads: Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
               out: Optional[Sequence[torch.Tensor]] = None) -> Tuple[List[torch.Tensor], torch.Tensor]:
    """``grads`` scaled by ``min(1, max_norm / (norm + 1e-6))`` and their norm.

    Writes to ``out`` (contiguous tensors of the same shapes and types, which overlap neither each
    other nor ``grads``; or the tensors of ``grads`` themselves) or to new tensors, and returns them.
    """
    return _ops().clip_grads(list(grads), max_norm, norm_type, None if out is None else list(out))


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` on the kernels: scales the ``grad`` of every parameter in
    place by ``min(1, max_norm / (norm + 1e-6))`` and returns the norm (0-d float32).

    The gradients are on one CUDA device and do not overlap: those that share memory, strided ones
    included, are refused (strided views that only interleave are not). ``error_if_nonfinite`` reads the
    norm on the host (so not under graph capture) and raises before anything is scaled."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [g for g in (p.grad for p in parameters) if g is not None]
    return _ops().clip_in_place(grads, max_norm, norm_type, error_if_nonfinite)


# ---------------------------------------------------------------------------- a torch world model
def _float32_under_autocast(x: torch.Tensor) -> torch.Tensor:
    """torch runs layer_norm in float32 under autocast; float64 stays (and is refused)."""
    return x.float() if x.dtype in (torch.bfloat16, torch.float16) and torch.is_autocast_enabled("cuda") else x


def _layer_norm_forward(module: torch.nn.LayerNorm, input: torch.Tensor) -> torch.Tensor:
    if input.dim() == 0 or input.shape[-1] != module.normalized_shape[0]:  # nothing else tells without weight and bias
        raise ValueError(f"input of shape {tuple(input.shape)} does not end in the norm's {module.normalized_shape[0]}")
    return layer_norm(_float32_under_autocast(input), module.weight, module.bias, module.eps)


def _watched(m: torch.nn.Module) -> bool:
    """Whether a hook wants to see the module called."""
    return bool(m._forward_pre_hooks or m._forward_hooks or m._backward_pre_hooks or m._backward_hooks
                or torch.nn.modules.module._has_any_global_hook())


def _modulates(m: torch.Tensor, x: torch.Tensor) -> bool:
    """Whether ``ada_layer_norm`` takes modulation ``m`` for ``x`` and gives what torch's products and sums
    would: a row of ``m`` for each or for consecutive rows of ``x``, and no type above that of ``x``."""
    if m.dtype != x.dtype and torch.promote_types(m.dtype, x.dtype) != x.dtype:
        return False
    ms, xs = m.shape, x.shape
    if ms == xs:
        return True
    if not 0 < len(ms) <= len(xs) or ms[-1] != xs[-1]:
        return False
    ms = (1,) * (len(xs) - len(ms)) + tuple(ms)
    d = len(ms) - 2
    while d >= 0 and ms[d] == 1:
        d -= 1
    return ms[:d + 1] == tuple(xs[:d + 1])


def _modulated_norm(norm: torch.nn.LayerNorm, x: torch.Tensor, shift: torch.Tensor,
                    scale: torch.Tensor) -> torch.Tensor:
    """``modulate(norm(x), shift, scale)``: in one pass where the kernel has the form and nothing else is asked
    of ``norm``, as a block's norms may have been hooked or changed since they were routed."""
    if _plain_norm(norm) and not _watched(norm):
        rows = _float32_under_autocast(x)
        if _modulates(shift, rows) and x.shape[-1] == norm.normalized_shape[0]:
            return ada_layer_norm(rows, shift, scale, norm.eps)
    return norm(x) * (1 + scale) + shift


def _conditional_block_forward(block: torch.nn.Module, x: torch.Tensor, c: torch.Tensor) -> torch.Tensor:
    """``ConditionalBlock.forward`` (reference ``lewm/module.py:105-111``)."""
    shift_a, scale_a, gate_a, shift_m, scale_m, gate_m = block.adaLN_modulation(c).chunk(6, dim=-1)
    x = x + gate_a * block.attn(_modulated_norm(block.norm1, x, shift_a, scale_a))
    return x + gate_m * block.mlp(_modulated_norm(block.norm2, x, shift_m, scale_m))


def _torch_norm(m: Any) -> bool:
    """A LayerNorm over the last dim that computes what torch's does."""
    return (isinstance(m, torch.nn.LayerNorm) and type(m).forward is torch.nn.LayerNorm.forward
            and len(m.normalized_shape) == 1)


def _plain_norm(m: Any) -> bool:
    """A LayerNorm over the last dim without an affine, as torch computes it or routed here."""
    own = getattr(m, "__dict__", {}).get("forward")
    return (_torch_norm(m) and m.weight is None and m.bias is None
            and (own is None or getattr(own, "func", None) is _layer_norm_forward))


# What a block's forward computes is read by running it on stand-ins that write down what is done to them,
# and compared with the formula that ``_conditional_block_forward`` computes.
class _Value:
    """How a value of a forward pass is made, as nested tuples; sums and products in one order."""

    __slots__ = ("made",)

    def __init__(self, *made: Any):
        self.made = made

    @staticmethod
    def _of(v: Any) -> tuple:
        if isinstance(v, _Value):
            return v.made
        if isinstance(v, (int, float)):
            return ("number", float(v))
        raise TypeError("not a value")

    def __add__(self, other: Any) -> "_Value":
        return _Value("+", *sorted((self.made, _Value._of(other)), key=repr))

    def __mul__(self, other: Any) -> "_Value":
        return _Value("*", *sorted((self.made, _Value._of(other)), key=repr))

    __radd__, __rmul__ = __add__, __mul__

    def chunk(self, chunks: int, dim: int = 0) -> tuple:
        return tuple(_Value("chunk", self.made, chunks, dim, i) for i in range(chunks))


class _Parts:
    """A block whose parts write down that they were called; it has nothing else, and nothing can be set."""

    __slots__ = ()

    def __getattr__(self, name: str):
        if name not in ("adaLN_modulation", "attn", "mlp", "norm1", "norm2"):
            raise AttributeError(name)
        return lambda v: _Value(name, _Value._of(v))


def _conditional_block_formula(block, x, c):
    """``ConditionalBlock.forward`` (reference ``lewm/module.py:105-111``)."""
    shift_a, scale_a, gate_a, shift_m, scale_m, gate_m = block.adaLN_modulation(c).chunk(6, dim=-1)
    x = x + gate_a * block.attn(block.norm1(x) * (1 + scale_a) + shift_a)
    return x + gate_m * block.mlp(block.norm2(x) * (1 + scale_m) + shift_m)


def _straight_line(f: Any, depth: int = 4) -> bool:
    """Whether ``f`` is a Python function that takes one way through its code, whatever else there is: no
    jumps, closures or handlers, nothing stored but its own variables, and of the globals only such functions."""
    if not isinstance(f, types.FunctionType) or depth == 0:
        return False
    code = f.__code__
    if code.co_freevars or code.co_cellvars or code.co_exceptiontable or f.__defaults__ or f.__kwdefaults__:
        return False
    for i in dis.get_instructions(code):
        if i.opcode in dis.hasjrel or i.opcode in dis.hasjabs or i.opname.startswith(("IMPORT", "MAKE", "DELETE")):
            return False
        if i.opname.startswith("STORE_") and not i.opname.startswith("STORE_FAST"):
            return False
        if i.opname == "LOAD_GLOBAL" and not _straight_line(f.__globals__.get(i.argval), depth - 1):
            return False
    return True


def _known_block(m: torch.nn.Module) -> bool:
    """An AdaLN conditional block whose forward is the known formula."""
    if (type(m).__name__ != "ConditionalBlock" or not all(hasattr(m, n) for n in ("adaLN_modulation", "attn", "mlp"))
            or not _plain_norm(getattr(m, "norm1", None)) or not _plain_norm(getattr(m, "norm2", None))
            or not _straight_line(type(m).forward)):
        return False
    forward = type(m).forward
    code = forward.__code__
    if code.co_argcount != 3 or code.co_kwonlyargcount or code.co_varnames[1:3] != ("x", "c") or \
            code.co_flags & (inspect.CO_VARARGS | inspect.CO_VARKEYWORDS | inspect.CO_GENERATOR | inspect.CO_COROUTINE):
        return False
    x, c = _Value("x"), _Value("c")
    try:
        got = forward(_Parts(), x, c)
    except Exception:  # it does something else than the formula needs
        return False
    return isinstance(got, _Value) and got.made == _conditional_block_formula(_Parts(), x, c).made


class B200TrainingNorms:
    """What ``install_training_norms`` routed: ``modules`` (names), and ``remove()`` to undo it."""

    def __init__(self, model: torch.nn.Module):
        self.modules: List[str] = []
        self._routed: List[torch.nn.Module] = []
        for name, m in model.named_modules():
            if "forward" in m.__dict__:  # routed already, by this or another install
                continue
            if _torch_norm(m):
                m.forward = functools.partial(_layer_norm_forward, m)
            elif _known_block(m):
                m.forward = functools.partial(_conditional_block_forward, m)
            else:
                continue
            self.modules.append(name)
            self._routed.append(m)

    def remove(self) -> None:
        for m in self._routed:
            if getattr(m.__dict__.get("forward"), "func", None) in (_layer_norm_forward, _conditional_block_forward):
                del m.__dict__["forward"]  # one set since then stays
        self._routed = []
        self.modules = []


def install_training_norms(model: torch.nn.Module) -> B200TrainingNorms:
    """Route every ``nn.LayerNorm`` over the last dim (not subclasses with a forward of their own) and
    every AdaLN ``ConditionalBlock`` of ``model`` whose forward computes the known formula (reference
    ``lewm/module.py:38-53,56-111,131-187,217-240``: predictor, projector heads, and the ViT encoder)
    through ``layer_norm`` and ``ada_layer_norm``, so that a training step of the world model runs their
    forward and backward passes on the B200 kernels. Parameters, state dict, hooks, type promotion and autocast behaviour stay as they are: under
    autocast the norms run in float32 as torch's do, and a block whose norms are hooked or were changed, or
    whose modulation broadcasts in a way the kernel has not, calls the norm and modulates by itself.
    The model's inputs must be on a CUDA device and not float64. Remove the routing to trace or export the
    model, or to take forward-mode derivatives."""
    return B200TrainingNorms(model)
