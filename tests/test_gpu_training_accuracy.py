"""Training norms on the GPU: rows whose mean is large beside their spread, and every pairing of types."""

import pytest
import torch

import lewm_flash_b200 as lf
from tests.test_gpu_training import BF16, DEV, F16, F32, activation, check_norm, randn
from tests.training_reference import U, assert_within

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------- constant rows, large offsets
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("rows,width", [(24, 1), (24, 3), (24, 40), (24, 192), (5000, 192), (24, 255), (5000, 300), (24, 384),
                                        (5000, 640), (24, 1011), (24, 1536), (24, 2047), (24, 3000), (24, 4097),
                                        (24, 6145), (24, 8192), (24, 12001), (24, 12008), (24, 16383), (24, 16384),
                                        (24, 20000), (24, 65535)])
def test_any_constant_row_gives_the_bias(rows, width, dtype):
    """A constant row c is a padding row: z is 0 and y the bias, to the bit. The first mean mu is off by
    m <= K steps of c (K u bounds a sum's relative error, tests/training_reference.py), so every c - mu is
    the same m steps; their sums are whole multiples of a step below 2^24 (width * K < 2^24 to the width of
    65535, where K is 104 + 64 steps), exact like their quotient by the width, which is what is taken off."""
    c = torch.tensor([0.1, 10.237, 1234.567, -1.0 / 3, 1999.9], device=DEV).to(dtype)
    x = c[torch.arange(rows, device=DEV) % 5][:, None].expand(rows, width).contiguous().requires_grad_(True)
    w, b = randn(width, seed=1, dtype=dtype), randn(width, seed=2, dtype=dtype)
    for eps in (1e-6, 1e-12):
        y = lf.layer_norm(x, w, b, eps=eps)
        assert torch.equal(y.detach(), b.expand(rows, -1))
    assert torch.equal(lf.ada_layer_norm(x, b, w).detach(), b.expand(rows, -1))
    per_row = [t.expand(rows, width).contiguous() for t in (b, w)]
    assert torch.equal(lf.ada_layer_norm(x, *per_row).detach(), per_row[0])


def offset_reference(x, gain, offset, eps, dy):
    """norm_reference for rows whose mean is taken in two steps: mu, then what is left of the mean of
    c = x - mu. c is exact where x lies within a factor of two of mu (else off by u |c|), so with K as there
      |e(mu)| <= K u mean|x| leaves c of size |x - mean| + |e(mu)|, and the mean's own error is (K + 2) u mean|c|;
      the variance is off by (2 K + 8) u mean(c^2);
    the backward pass starts from the mean rounded to float32, u |mean| more."""
    x, gain, offset, dy = x.double(), gain.double(), offset.double(), dy.double()
    n = x.shape[-1]
    K = (56 if n <= 16384 else 104 + n / 1024) * U
    mu = x.mean(-1, keepdim=True)
    xc = x - mu
    var = (xc * xc).mean(-1, keepdim=True)
    rs = 1.0 / torch.sqrt(var + eps)
    z = xc * rs
    c = xc.abs() + K * x.abs().mean(-1, keepdim=True) + U * mu.abs()
    e_mu = (K + 2 * U) * c.mean(-1, keepdim=True)
    e_rs = 0.5 * (2 * K + 8 * U) * (c * c).mean(-1, keepdim=True) * rs * rs + 3 * U
    e_z = rs * (e_mu + 2 * U * c) + z.abs() * (e_rs + 2 * U)
    y = z * gain + offset
    e_y = e_z * gain.abs() + 3 * U * ((z * gain).abs() + offset.abs())
    e_z = e_z + rs * U * mu.abs()
    d = dy * gain
    m1, m2 = d.mean(-1, keepdim=True), (d * z).mean(-1, keepdim=True)
    dx = rs * (d - m1 - z * m2)
    e_m1 = K * d.abs().mean(-1, keepdim=True)
    e_m2 = K * (d * z).abs().mean(-1, keepdim=True) + (d.abs() * e_z).mean(-1, keepdim=True)
    size = d.abs() + m1.abs() + (z * m2).abs()
    e_dx = rs * (5 * U * size + e_m1 + z.abs() * e_m2 + e_z * m2.abs()) + dx.abs() * (e_rs + 2 * U)
    return y, e_y, dx, e_dx


@pytest.mark.parametrize("rows,width", [(30, 48), (30, 192), (5000, 192), (30, 384), (30, 1011), (30, 1536), (30, 4096),
                                        (30, 8192), (6, 20000), (6, 20003)])
@pytest.mark.parametrize("offset,spread", [(1000.0, 1e-2), (37.0, 1e-4), (-3e5, 1.0)])
def test_small_spread_on_a_large_offset(rows, width, offset, spread):
    x = randn(rows, width, seed=1, scale=spread, offset=offset).requires_grad_(True)
    w, b = randn(width, seed=2, scale=0.2, offset=1.0), randn(width, seed=3)
    dy = randn(rows, width, seed=4)
    y = lf.layer_norm(x, w, b)
    (dx,) = torch.autograd.grad(y, x, dy)
    want, e_y, want_dx, e_dx = offset_reference(x.detach(), w, b, 1e-5, dy)
    assert_within(y.detach(), want, e_y, F32, "y")
    assert_within(dx, want_dx, e_dx, F32, "dx")


def test_squares_that_overflow_stay_finite():
    """x of 1e30: the variance is infinite in float32, z is 0 and y the bias, as torch's layer_norm has it."""
    x = randn(8, 192, seed=1, scale=1e30)
    x[3] = 1e30
    w, b = randn(192, seed=2), randn(192, seed=3)
    assert torch.equal(lf.layer_norm(x, w, b)[[0, 1, 2, 4, 5, 6, 7]], b.expand(7, -1))
    assert torch.equal(lf.layer_norm(x[3:4], w, b), b.expand(1, -1))
    wide = randn(3, 20000, seed=4, scale=1e30)
    assert not lf.layer_norm(wide).any()


# ---------------------------------------------------------------------------- every pairing of types
@pytest.mark.parametrize("dtype,ctype", [(F32, BF16), (F32, F16), (BF16, F16), (F16, BF16), (BF16, BF16), (F16, F32)],
                         ids=["f32-bf16", "f32-f16", "bf16-f16", "f16-bf16", "bf16", "f16-f32"])
@pytest.mark.parametrize("batch,tokens,width", [(1, 1, 192), (300, 3, 192), (2000, 3, 192), (1700, 3, 384), (7, 5, 33),
                                                (1000, 5, 70), (40, 15, 2050), (9, 40, 640), (5000, 1, 154),
                                                (7, 30, 4100), (20, 3, 8192), (9, 4, 10008), (3, 2, 16385)])
@pytest.mark.parametrize("shared", [False, True], ids=["per_token", "per_sequence"])
def test_ada_layer_norm_of_mixed_types(batch, tokens, width, shared, dtype, ctype):
    """float32 rows with 16-bit modulation are what a float32 model gives under autocast."""
    x = activation(batch * tokens, width, dtype).view(batch, tokens, width).requires_grad_(True)
    mod = randn(batch, 1 if shared else tokens, 6 * width, seed=3, scale=0.4, dtype=ctype)
    shift, scale = (t.requires_grad_(True) for t in mod.chunk(6, -1)[:2])
    dy = randn(batch, tokens, width, seed=7, scale=0.1, dtype=dtype)
    y = lf.ada_layer_norm(x, shift, scale)
    dx, dshift, dscale = torch.autograd.grad(y, (x, shift, scale), dy)
    assert y.dtype == dtype and dshift.dtype == dscale.dtype == ctype
    check_norm(x, scale, shift, 1e-6, True, tokens if shared else 1, y.detach(), dy, dx, dscale, dshift)
