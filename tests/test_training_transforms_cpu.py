"""Training operators, no GPU: callers that the kernels would answer wrongly are refused by name, before
anything else is looked at."""

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx

import lewm_flash_b200 as lf

z = torch.zeros


# ---------------------------------------------------------------------------- forward mode
@pytest.mark.parametrize("call", [
    lambda d: lf.layer_norm(d(3, 8)),
    lambda d: lf.layer_norm(z(3, 8), d(8)),
    lambda d: lf.layer_norm(z(3, 8), z(8), d(8)),
    lambda d: lf.ada_layer_norm(d(3, 8), z(8), z(8)),
    lambda d: lf.ada_layer_norm(z(3, 8), d(8), z(8)),
    lambda d: lf.ada_layer_norm(z(3, 8), z(8), d(8)),
    lambda d: lf.grad_norm([z(3), d(3)]),
    lambda d: lf.clip_grads([d(3)], 1.0),
    lambda d: lf.clip_grads([z(3)], 1.0, out=[d(3)]),
])
def test_forward_mode_is_refused(call):
    with fwd.dual_level():
        def dual(*shape):
            return fwd.make_dual(z(*shape), torch.ones(*shape))

        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):  # has tangents all the same
            call(dual)
        with pytest.raises(ValueError, match="need a CUDA device"):
            call(z)


def test_forward_mode_of_a_routed_model_is_refused():
    model = torch.nn.Sequential(torch.nn.LayerNorm(8))
    lf.install_training_norms(model)
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        model(fwd.make_dual(z(3, 8), z(3, 8)))


# ---------------------------------------------------------------------------- tracers
@pytest.mark.parametrize("trace", [
    lambda f, x: torch.jit.trace(f, (x,), check_trace=False),
    lambda f, x: make_fx(f)(x),
    lambda f, x: make_fx(f, tracing_mode="fake")(x),
    lambda f, x: make_fx(f, tracing_mode="symbolic")(x),
    lambda f, x: make_fx(f, pre_dispatch=True)(x),
], ids=["jit", "make_fx", "fake", "symbolic", "pre_dispatch"])
@pytest.mark.parametrize("call", [lambda x: lf.layer_norm(x), lambda x: lf.ada_layer_norm(x, z(8), z(8)),
                                  lambda x: lf.grad_norm([x]), lambda x: lf.clip_grads([x], 1.0)[1],
                                  lambda x: x + lf.layer_norm(z(8))])
def test_tracing_is_refused(call, trace):
    with pytest.raises(NotImplementedError, match="cannot be traced"):
        trace(call, z(3, 8))
    with pytest.raises(ValueError, match="need a CUDA device"):
        call(z(3, 8))


# ---------------------------------------------------------------------------- function transforms, subclasses
TRANSFORMS = {
    "vmap": lambda f: torch.vmap(f)(z(2, 3, 8)),
    "grad": lambda f: torch.func.grad(lambda t: f(t).sum())(z(3, 8)),
    "jvp": lambda f: torch.func.jvp(f, (z(3, 8),), (z(3, 8),)),
    "jacrev": lambda f: torch.func.jacrev(f)(z(3, 8)),
    "jacfwd": lambda f: torch.func.jacfwd(f)(z(3, 8)),
    "functionalize": lambda f: torch.func.functionalize(f)(z(3, 8)),
}
CALLS = [lambda x: lf.layer_norm(x), lambda x: lf.layer_norm(z(3, 8), x[0]), lambda x: lf.ada_layer_norm(x, z(8), z(8)),
         lambda x: lf.ada_layer_norm(z(3, 8), z(3, 8), x), lambda x: lf.grad_norm([z(2), x]),
         lambda x: lf.clip_grads([x], 1.0)[1], lambda x: lf.clip_grads([z(8)], 1.0, out=[x[0]])[1]]


@pytest.mark.parametrize("transform", list(TRANSFORMS.values()), ids=list(TRANSFORMS))
@pytest.mark.parametrize("call", CALLS)
def test_function_transforms_are_refused_by_name(call, transform):
    with pytest.raises(NotImplementedError, match="torch.func"):
        transform(call)


def test_function_transforms_around_plain_tensors_are_fine():
    plain = z(3, 8)

    def f(x):
        lf.layer_norm(plain)
        return x

    for transform in TRANSFORMS.values():
        with pytest.raises(ValueError, match="need a CUDA device"):
            transform(f)


def test_dispatching_subclasses_are_refused_by_name():
    class Wrapped(torch.Tensor):
        __torch_function__ = torch._C._disabled_torch_function_impl

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            return NotImplemented

    x = torch.Tensor._make_subclass(Wrapped, z(3, 8))
    with pytest.raises(NotImplementedError, match="__torch_dispatch__"):
        lf.layer_norm(x)
    with pytest.raises(NotImplementedError, match="__torch_dispatch__"):
        lf.clip_grads([z(3), x], 1.0)


def test_subclasses_and_modes_see_the_norms():
    class Recorder(torch.Tensor):
        seen = []

        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            cls.seen.append(func)
            return "answered"

    r = z(3, 8).as_subclass(Recorder)
    assert lf.layer_norm(r) == "answered" and lf.layer_norm(z(3, 8), r) == "answered"
    assert lf.ada_layer_norm(z(3, 8), z(8), r) == "answered"
    assert Recorder.seen == [lf.layer_norm, lf.layer_norm, lf.ada_layer_norm]

    class Mode(torch.overrides.TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func if func in (lf.layer_norm, lf.ada_layer_norm) else func(*args, **(kwargs or {}))

    with Mode():
        assert lf.layer_norm(z(3, 8)) is lf.layer_norm
    with torch.device("cpu"), pytest.raises(ValueError, match="need a CUDA device"):
        lf.layer_norm(z(3, 8))
