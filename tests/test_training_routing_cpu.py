"""install_training_norms, no GPU: which modules are routed, and that routed ones do what they did. The
operators are replaced by plain torch forms where a routed module runs."""

import pytest
import torch

import lewm_flash_b200 as lf
from lewm_flash_b200 import training
from tests import training_reference
from tests.training_reference import modulate

FLAG = False


def block_class(forward, name="ConditionalBlock"):
    return type(name, (training_reference.ConditionalBlock,), {"forward": forward})


# ---------------------------------------------------------------------------- which blocks
def reference_spelling(self, x, c):
    shift_msa, scale_msa, gate_msa, shift_mlp, scale_mlp, gate_mlp = self.adaLN_modulation(c).chunk(6, dim=-1)
    x = x + gate_msa * self.attn(modulate(self.norm1(x), shift_msa, scale_msa))
    x = x + gate_mlp * self.mlp(modulate(self.norm2(x), shift_mlp, scale_mlp))
    return x


def inlined(self, x, c):
    m = self.adaLN_modulation(c).chunk(6, -1)
    a, b, d, e, f, g = m
    h = self.norm1(x)
    x = self.attn(a + (b + 1) * h) * d + x
    return self.mlp((1.0 + f) * self.norm2(x) + e) * g + x


@pytest.mark.parametrize("forward", [reference_spelling, inlined])
def test_blocks_of_the_known_formula_are_routed(forward):
    block = block_class(forward)(8, 1, 8, 8)
    assert lf.install_training_norms(block).modules == ["", "attn.norm", "mlp.0", "norm1", "norm2"]


def scale_first(self, x, c):
    ka, sa, ga, km, sm, gm = self.adaLN_modulation(c).chunk(6, dim=-1)
    x = x + ga * self.attn(modulate(self.norm1(x), sa, ka))
    return x + gm * self.mlp(modulate(self.norm2(x), sm, km))


def no_residual(self, x, c):
    sa, ka, ga, sm, km, gm = self.adaLN_modulation(c).chunk(6, dim=-1)
    x = ga * self.attn(modulate(self.norm1(x), sa, ka))
    return x + gm * self.mlp(modulate(self.norm2(x), sm, km))


def first_residual_twice(self, x, c):
    sa, ka, ga, sm, km, gm = self.adaLN_modulation(c).chunk(6, dim=-1)
    h = x + ga * self.attn(modulate(self.norm1(x), sa, ka))
    return x + gm * self.mlp(modulate(self.norm2(h), sm, km))


def scale_without_one(self, x, c):
    sa, ka, ga, sm, km, gm = self.adaLN_modulation(c).chunk(6, dim=-1)
    x = x + ga * self.attn(self.norm1(x) * ka + sa)
    return x + gm * self.mlp(self.norm2(x) * km + sm)


def other_chunks(self, x, c):
    sa, ka, ga, sm, km, gm = self.adaLN_modulation(c).chunk(6, dim=1)
    x = x + ga * self.attn(modulate(self.norm1(x), sa, ka))
    return x + gm * self.mlp(modulate(self.norm2(x), sm, km))


def norms_swapped(self, x, c):
    sa, ka, ga, sm, km, gm = self.adaLN_modulation(c).chunk(6, dim=-1)
    x = x + ga * self.attn(modulate(self.norm2(x), sa, ka))
    return x + gm * self.mlp(modulate(self.norm1(x), sm, km))


def otherwise_when_evaluated(self, x, c):
    if not self.training:
        return x
    return reference_spelling(self, x, c)


def otherwise_by_a_global(self, x, c):
    return reference_spelling(self, x, c) if not FLAG else x


def counted(self, x, c):
    self.calls = 1
    sa, ka, ga, sm, km, gm = self.adaLN_modulation(c).chunk(6, dim=-1)
    x = x + ga * self.attn(modulate(self.norm1(x), sa, ka))
    return x + gm * self.mlp(modulate(self.norm2(x), sm, km))


def through_torch(self, x, c):
    sa, ka, ga, sm, km, gm = self.adaLN_modulation(c).chunk(6, dim=-1)
    x = torch.addcmul(x, ga, self.attn(modulate(self.norm1(x), sa, ka)))
    return x + gm * self.mlp(modulate(self.norm2(x), sm, km))


def more_arguments(self, x, c, mask=None):
    return reference_spelling(self, x, c)


def other_names(self, x, cond):
    return reference_spelling(self, x, cond)


def half_modulate(x, shift, scale):
    return x * (1 + 0.5 * scale) + shift


def by_another_modulate(self, x, c):
    sa, ka, ga, sm, km, gm = self.adaLN_modulation(c).chunk(6, dim=-1)
    x = x + ga * self.attn(half_modulate(self.norm1(x), sa, ka))
    return x + gm * self.mlp(half_modulate(self.norm2(x), sm, km))


OTHERS = [scale_first, no_residual, first_residual_twice, scale_without_one, other_chunks, norms_swapped,
          otherwise_when_evaluated, otherwise_by_a_global, counted, through_torch, more_arguments, other_names,
          by_another_modulate, torch.no_grad()(reference_spelling), lambda self, x, c: x]


@pytest.mark.parametrize("forward", OTHERS, ids=[f.__name__ for f in OTHERS])
def test_blocks_with_a_forward_of_their_own_are_left_alone(forward):
    block = block_class(forward)(8, 1, 8, 8)
    assert lf.install_training_norms(block).modules == ["attn.norm", "mlp.0", "norm1", "norm2"]
    assert "forward" not in block.__dict__ and "calls" not in block.__dict__


def test_blocks_with_norms_of_their_own_are_left_alone():
    class Scaled(torch.nn.LayerNorm):
        def forward(self, x):
            return 2 * super().forward(x)

    for norm in (Scaled(8, elementwise_affine=False), torch.nn.LayerNorm(8), torch.nn.LayerNorm((3, 8), elementwise_affine=False),
                 torch.nn.Identity()):
        block = block_class(reference_spelling)(8, 1, 8, 8)
        block.norm2 = norm
        assert "" not in lf.install_training_norms(block).modules
    block = block_class(reference_spelling)(8, 1, 8, 8)
    block.norm1.forward = lambda x: 3 * x
    assert lf.install_training_norms(block).modules == ["attn.norm", "mlp.0", "norm2"]


# ---------------------------------------------------------------------------- routed blocks
def plain_layer_norm(x, weight=None, bias=None, eps=1e-5):
    return torch.nn.functional.layer_norm(x, x.shape[-1:], weight, bias, eps)


def plain_ada_layer_norm(x, shift, scale, eps=1e-6):
    """The kernel's contract: modulation of x's shape, or of size 1 in dims right before the last; x's type."""
    m = (1,) * (x.dim() - shift.dim()) + tuple(shift.shape)
    d = x.dim() - 2
    while d >= 0 and m[d] == 1:
        d -= 1
    assert m == tuple(x.shape) or (m[-1] == x.shape[-1] and m[:d + 1] == tuple(x.shape)[:d + 1])
    y = plain_layer_norm(x.double(), eps=eps) * (1 + scale.double()) + shift.double()
    return y.to(x.dtype)


@pytest.fixture
def plain_forms(monkeypatch):
    """The operators in plain torch, so that routed modules run on the CPU; counts their calls."""
    calls = {"layer_norm": 0, "ada_layer_norm": 0}

    def counting(name, f):
        def g(*args, **kwargs):
            calls[name] += 1
            return f(*args, **kwargs)
        return g

    monkeypatch.setattr(training, "layer_norm", counting("layer_norm", plain_layer_norm))
    monkeypatch.setattr(training, "ada_layer_norm", counting("ada_layer_norm", plain_ada_layer_norm))
    return calls


def a_block():
    torch.manual_seed(0)
    return training_reference.ConditionalBlock(16, 2, 8, 32)


def close(a, b):
    return torch.allclose(a, b, rtol=1e-5, atol=1e-5)


def test_block_calls_each_norm_once_in_one_pass(plain_forms):
    block, x, c = a_block(), torch.randn(2, 3, 16), torch.randn(2, 3, 16)
    want = block(x, c)
    lf.install_training_norms(block)
    assert close(block(x, c), want)
    assert plain_forms == {"layer_norm": 2, "ada_layer_norm": 2}  # attn.norm and mlp.0


@pytest.mark.parametrize("register", [
    lambda n, f: n.register_forward_hook(lambda m, i, o: f(o)),
    lambda n, f: n.register_forward_pre_hook(lambda m, i: f(i[0].sin())),  # a norm undoes a factor
    lambda n, f: n.register_forward_hook(lambda m, i, k, o: f(o), with_kwargs=True),
    lambda n, f: n.register_full_backward_hook(lambda m, gi, go: (f(gi[0]),)),
    lambda n, f: n.register_full_backward_pre_hook(lambda m, go: (f(go[0]),)),
], ids=["forward", "forward_pre", "forward_kwargs", "backward", "backward_pre"])
@pytest.mark.parametrize("when", ["before", "after"])
def test_hooks_on_a_blocks_norms_run(plain_forms, register, when):
    """Hooks that double what they see, on both norms, set before or after routing."""
    block, x, c = a_block(), torch.randn(2, 3, 16, requires_grad=True), torch.randn(2, 3, 16)
    calls = []

    def double(t):
        calls.append(t.shape)
        return 2 * t

    def run():
        return block(x, c), *torch.autograd.grad(block(x, c).square().sum(), x)

    plain = run()
    if when == "after":
        handle = lf.install_training_norms(block)
    hooks = [register(n, double) for n in (block.norm1, block.norm2)]
    if when == "before":
        handle = lf.install_training_norms(block)
    got, seen = run(), len(calls)
    handle.remove()
    want = run()
    assert len(calls) == 2 * seen and seen >= 2
    assert all(close(p, q) for p, q in zip(got, want)) and not close(want[1], plain[1])
    for h in hooks:
        h.remove()


def test_hooks_on_all_modules_see_a_blocks_norms(plain_forms):
    block, x, c = a_block(), torch.randn(2, 3, 16), torch.randn(2, 3, 16)
    lf.install_training_norms(block)
    seen = []
    hook = torch.nn.modules.module.register_module_forward_hook(lambda m, i, o: seen.append(m))
    try:
        block(x, c)
    finally:
        hook.remove()
    assert block.norm1 in seen and block.norm2 in seen


def test_a_blocks_norms_may_change_after_routing(plain_forms):
    block, x, c = a_block(), torch.randn(2, 3, 16), torch.randn(2, 3, 16)
    handle = lf.install_training_norms(block)
    block.norm1 = torch.nn.LayerNorm(16)  # with an affine
    with torch.no_grad():
        block.norm1.weight.mul_(3.0)
    block.norm2.eps = 0.5
    got = block(x, c)
    handle.remove()
    assert close(got, block(x, c))
    block = a_block()
    lf.install_training_norms(block)
    block.norm2 = torch.nn.Identity()
    got = block(x, c)
    assert close(got, type(block).forward(block, x, c))


@pytest.mark.parametrize("x,c", [
    ((2, 3, 16), (3, 16)),        # one window's conditioning for all
    ((2, 3, 16), (1, 3, 16)),
    ((2, 3, 16), (16,)),
    ((2, 3, 16), (2, 1, 16)),
    ((2, 3, 16), (1, 1, 16)),
    ((2, 1, 16), (2, 3, 16)),     # the result grows
    ((1, 3, 16), (2, 3, 16)),
    ((2, 1, 16), (2, 1, 16)),
])
def test_conditioning_of_any_shape_that_broadcasts(plain_forms, x, c):
    block, x, c = a_block(), torch.randn(x), torch.randn(c)
    want = block(x, c)
    lf.install_training_norms(block)
    got = block(x, c)
    assert got.shape == want.shape and close(got, want)


class Cast(torch.nn.Module):
    """Keeps a block's parts in float32 behind a stream of another type."""

    def __init__(self, inner, out=None):
        super().__init__()
        self.inner, self.out = inner, out

    def forward(self, x):
        y = self.inner(x.float())
        return y if self.out is None else y.to(self.out)


@pytest.mark.parametrize("stream", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mod", [torch.float32, torch.bfloat16, torch.float16])
def test_types_promote_as_they_did(plain_forms, stream, mod):
    """A modulation type above that of x lifts the result, as in torch: float32 stays float32 behind bf16 rows."""
    block = a_block()
    seen = []
    block.attn, block.mlp = Cast(block.attn), Cast(block.mlp)
    block.adaLN_modulation = Cast(block.adaLN_modulation, mod)
    for m in (block.attn, block.mlp):
        m.register_forward_pre_hook(lambda m, i: seen.append(i[0].dtype))
    x, c = torch.randn(2, 3, 16).to(stream), torch.randn(2, 3, 16)
    want = block(x, c)
    lf.install_training_norms(block)
    got = block(x, c)
    assert got.dtype == want.dtype and seen[:2] == seen[2:]
    assert torch.allclose(got.float(), want.float(), rtol=0.05, atol=0.05)  # a few roundings to 2^-8 of values of 4
    assert seen[0] == torch.promote_types(stream, mod)


# ---------------------------------------------------------------------------- what torch's modules refuse
@pytest.mark.parametrize("affine", [False, True])
@pytest.mark.parametrize("shape", [(3, 7), (3, 16, 1), ()])
def test_rows_of_another_width_stay_refused(plain_forms, affine, shape):
    norm = torch.nn.LayerNorm(16, elementwise_affine=affine)
    with pytest.raises(RuntimeError):
        norm(torch.zeros(shape))
    lf.install_training_norms(norm)
    with pytest.raises(ValueError, match="does not end in the norm's 16"):
        norm(torch.zeros(shape))


def test_blocks_of_another_width_stay_refused(plain_forms):
    block = a_block()
    block.norm1 = torch.nn.LayerNorm(8, elementwise_affine=False)
    x, c = torch.randn(2, 3, 16), torch.randn(2, 3, 16)
    with pytest.raises(RuntimeError):
        block(x, c)
    lf.install_training_norms(block)
    with pytest.raises(ValueError, match="does not end in the norm's 8"):
        block(x, c)


def test_float64_is_not_rounded_under_autocast(monkeypatch):
    """torch keeps float64 there; the kernels have no float64."""
    monkeypatch.setattr(torch, "is_autocast_enabled", lambda device=None: True)
    norm, block = torch.nn.LayerNorm(8), a_block().double()
    lf.install_training_norms(norm), lf.install_training_norms(block)
    with pytest.raises(ValueError, match="must be float32"):
        norm(torch.zeros(3, 8, dtype=torch.float64))
    with pytest.raises(ValueError, match="must be float32"):
        block(*torch.zeros(2, 2, 3, 16, dtype=torch.float64))
    with pytest.raises(ValueError, match="need a CUDA device"):
        norm(torch.zeros(3, 8, dtype=torch.bfloat16))


def test_removal_leaves_forwards_set_since():
    model = torch.nn.Sequential(torch.nn.LayerNorm(8), torch.nn.LayerNorm(8))
    handle = lf.install_training_norms(model)
    own = model[0].forward = lambda x: 3 * x
    handle.remove()
    assert model[0].__dict__["forward"] is own and "forward" not in model[1].__dict__


class Doubled(torch.nn.Module):
    def forward(self, x):
        return 2 * x


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_models_with_scripted_parts_are_routed_around_them():
    model = torch.nn.Sequential(torch.jit.script(Doubled()), torch.jit.trace(Doubled(), torch.zeros(2)),
                                torch.jit.script(torch.nn.LayerNorm(8)), torch.nn.LayerNorm(8))
    assert lf.install_training_norms(model).modules == ["3"]


def test_routed_modules_take_their_arguments_by_name(plain_forms):
    norm, block = torch.nn.LayerNorm(16), a_block()
    x, c = torch.randn(2, 3, 16), torch.randn(2, 3, 16)
    want = norm(input=x), block(x, c=c), block(c=c, x=x)
    lf.install_training_norms(norm), lf.install_training_norms(block)
    assert all(close(p, q) for p, q in zip((norm(input=x), block(x, c=c), block(c=c, x=x)), want))
