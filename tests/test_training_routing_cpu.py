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
