"""Training operators on the GPU: the gradients' memory, and autograd's less usual callers."""

import pytest
import torch

import lewm_flash_b200 as lf
from tests.test_gpu_training import BF16, DEV, F32, activation, randn

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------- whose memory a gradient is
@pytest.mark.parametrize("shape", [(300, 3, 192), (6, 64), (40, 1030)])
def test_gradients_of_a_shift_per_row_share_no_memory(shape):
    """The shift's gradient is the output's gradient, in memory that nobody else holds: after two
    accumulated passes each is the sum of two equal addends (exact), and the caller's own is as it was."""
    x, scale = randn(*shape, seed=1), randn(*shape, seed=2, scale=0.3)
    shifts = [randn(*shape, seed=s).requires_grad_(True) for s in (3, 4)]
    g = randn(*shape, seed=5)
    before = g.clone()
    for _ in range(2):
        (lf.ada_layer_norm(x, shifts[0], scale) + lf.ada_layer_norm(x, shifts[1], scale)).backward(g)
    assert len({t.data_ptr() for t in (shifts[0].grad, shifts[1].grad, g)}) == 3
    assert torch.equal(g, before)
    assert torch.equal(shifts[0].grad, 2 * before) and torch.equal(shifts[1].grad, 2 * before)
    norm = lf.clip_grad_norm_(shifts, 1.0)  # refuses gradients that overlap
    assert norm > 1.0 and torch.equal(g, before)


@pytest.mark.parametrize("retain", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradient_of_a_shift_per_row_from_an_operator_behind(dtype, retain):
    """The output's gradient comes from an operator that keeps nothing of it, or, retained, is y.grad too."""
    x, scale, k = (randn(50, 192, seed=s, dtype=dtype) for s in (1, 2, 3))
    shift = randn(50, 192, seed=4, dtype=dtype).requires_grad_(True)
    for n in (1, 2):
        y = lf.ada_layer_norm(x, shift, scale)
        if retain:
            y.retain_grad()
        (y * k).sum().backward()
        assert torch.equal(shift.grad, n * k)
        if retain:
            assert torch.equal(y.grad, k) and y.grad.data_ptr() != shift.grad.data_ptr()
    with torch.no_grad():
        shift.grad.zero_()
    assert k.any()


def test_gradient_of_a_shift_per_row_seen_by_hooks():
    """Hooks that keep the gradient they are shown keep it for themselves."""
    x, scale, k = (randn(50, 192, seed=s) for s in (1, 2, 3))
    shift = randn(50, 192, seed=4).requires_grad_(True)
    y = lf.ada_layer_norm(x, shift, scale)
    kept = []
    y.register_hook(lambda g: kept.append(g))
    y.grad_fn.register_hook(lambda gi, go: kept.append(go[0]))
    shift.register_hook(lambda g: kept.append(g.clone()))
    (y * k).sum().backward()
    with torch.no_grad():
        shift.grad.mul_(3.0)
    assert len(kept) == 3 and all(torch.equal(g, k) for g in kept)


def test_returned_gradient_of_a_shift_per_row_is_not_the_given_one():
    x, scale = randn(20, 64, seed=1), randn(20, 64, seed=2)
    shift, g = randn(20, 64, seed=3).requires_grad_(True), randn(20, 64, seed=4)
    (d,) = torch.autograd.grad(lf.ada_layer_norm(x, shift, scale), shift, g)
    assert torch.equal(d, g) and d.data_ptr() != g.data_ptr()
    before = g.clone()
    lf.clip_grads([d], 0.1, out=[d])
    assert torch.equal(g, before)


# ---------------------------------------------------------------------------- forward mode
def test_forward_mode_through_a_backward_pass_is_refused():
    """A tangent on the output's gradient (forward over reverse) would be dropped."""
    import torch.autograd.forward_ad as fwd

    x = randn(4, 32).requires_grad_(True)
    y = lf.layer_norm(x)
    with fwd.dual_level():
        dy = fwd.make_dual(randn(4, 32, seed=1), randn(4, 32, seed=2))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, dy)


def test_forward_mode_is_refused_on_the_gpu():
    import torch.autograd.forward_ad as fwd

    x, w = randn(4, 32), randn(32)
    with fwd.dual_level():
        for args in ((fwd.make_dual(x, x), w), (x, fwd.make_dual(w, w))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                lf.layer_norm(*args)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            lf.grad_norm([x, fwd.make_dual(x, x)])
        lf.layer_norm(x, w)  # nothing dual: as ever


# ---------------------------------------------------------------------------- tracers
def test_tracing_is_refused_on_the_gpu():
    """A tracer does not see the kernels and would record their output as a constant."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x, w = randn(4, 32), randn(32)
    for call in (lambda t: lf.layer_norm(t, w), lambda t: lf.ada_layer_norm(t, w, w), lambda t: lf.grad_norm([t]),
                 lambda t: lf.clip_grads([t], 0.1)[0][0]):
        for trace in (lambda f: torch.jit.trace(f, (x,), check_trace=False), lambda f: make_fx(f)(x),
                      lambda f: make_fx(f, tracing_mode="fake")(x), lambda f: make_fx(f, pre_dispatch=True)(x)):
            with pytest.raises(NotImplementedError, match="trac"):
                trace(call)
        call(x)  # the tracer is gone


def test_tracing_a_backward_pass_is_refused():
    from torch.fx.experimental.proxy_tensor import make_fx

    x = randn(4, 32).requires_grad_(True)
    y = lf.layer_norm(x)
    with pytest.raises(NotImplementedError, match="trac"):
        make_fx(lambda g: torch.autograd.grad(y, x, g, retain_graph=True)[0])(randn(4, 32, seed=1))


# ---------------------------------------------------------------------------- lazily negated gradients
@pytest.mark.parametrize("rows,width", [(50, 1), (50, 192), (9, 20000)])
def test_lazily_negated_output_gradient(rows, width):
    x, w, b = randn(rows, width, seed=1), randn(width, seed=2), randn(width, seed=3)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    dy = randn(rows, width, seed=4)
    y = lf.layer_norm(*leaves)
    want = torch.autograd.grad(y, leaves, -dy, retain_graph=True)
    got = torch.autograd.grad(y, leaves, torch._neg_view(dy))
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    shift, scale = (randn(rows, width, seed=s).requires_grad_(True) for s in (5, 6))
    y = lf.ada_layer_norm(x, shift, scale)
    want = torch.autograd.grad(y, (x, shift, scale), -dy, retain_graph=True)
    got = torch.autograd.grad(y, (x, shift, scale), torch._neg_view(dy))
    assert all(torch.equal(p, q) and not p.is_neg() for p, q in zip(got, want))


# ---------------------------------------------------------------------------- function transforms, subclasses
def test_batched_output_gradients_are_refused():
    x = randn(4, 32).requires_grad_(True)
    y = lf.layer_norm(x)
    with pytest.raises(NotImplementedError, match="torch.func"):
        torch.autograd.grad(y, x, randn(3, 4, 32, seed=1), is_grads_batched=True)


def test_tensor_subclasses_stay():
    class Named(torch.Tensor):
        pass

    x, w = activation(20, 192, F32), randn(192, seed=2)
    y = lf.layer_norm(x.as_subclass(Named), w)
    assert type(y) is Named and torch.equal(y.as_subclass(torch.Tensor), lf.layer_norm(x, w))
    y = lf.ada_layer_norm(x, w.as_subclass(Named), w)
    assert type(y) is Named and torch.equal(y.as_subclass(torch.Tensor), lf.ada_layer_norm(x, w, w))
    assert type(lf.layer_norm(torch.nn.Parameter(x), w)) is torch.Tensor


# ---------------------------------------------------------------------------- a routed model
def test_routed_model_saved_loaded_and_run_under_autograds_modes():
    import io

    from tests.training_reference import TinyPredictor

    torch.manual_seed(0)
    model = TinyPredictor().to(DEV)
    lf.install_training_norms(model)
    x, c = randn(5, 3, 64, seed=1).requires_grad_(True), randn(5, 3, 64, seed=2)

    def grad():
        (g,) = torch.autograd.grad(model(x, c).square().sum(), x)
        return g

    want = grad()
    with torch.autograd.set_detect_anomaly(True):
        assert torch.equal(grad(), want)
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t) or t.clone(), lambda t: t):
        y = model(x, c)
    assert torch.equal(torch.autograd.grad(y.square().sum(), x)[0], want) and packed
    buf = io.BytesIO()
    torch.save(model, buf)
    buf.seek(0)
    loaded = torch.load(buf, weights_only=False)
    assert torch.equal(loaded(x, c), model(x, c))
    with torch.no_grad():
        for p in loaded.parameters():
            p.zero_()
    assert not loaded(x, c).any() and model(x, c).any()  # its own parameters
