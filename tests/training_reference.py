"""Plain 64-bit forms of the training operators with bounds on a float32 kernel's error, and a small
torch restatement of the reference's predictor block (``lewm/module.py:38-111``) for tests."""

import math

import torch

U = 2.0 ** -24  # half a float32 step, relative


def half_step(dtype):
    """Largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def norm_reference(x, gain, offset, eps, dy=None):
    """Layer norm of x (R, n) with gain, offset broadcastable to it, in float64: a dict of y, dx, the
    per-row products whose sums are the parameter gradients (pz = dy z, p1 = dy), and for each an
    elementwise bound on the error of a float32 evaluation.

    The bound, with u = 2^-24: a row sum takes at most 16 adds in a thread (64 a thread on rows past
    16384 values), 5 in a warp and 32 across warps, so K = 16 + 5 + 32 + 3 <= 56 roundings (104) of a sum
    of magnitudes S give an error <= K u S. So
      |e(mu)| <= K u mean|x|
      e(var)/var <= (K + 4) u + e(mu)^2 / var, and rs has half of it + 3 u
      |e(z)| <= rs (e(mu) + u |x - mu|) + |z| (e(rs)/rs + 2 u)
    and products, sums and the final combination add one rounding each."""
    x = x.double()
    n = x.shape[-1]
    K = (56 if n <= 16384 else 104 + n / 1024) * U
    mu = x.mean(-1, keepdim=True)
    xc = x - mu
    var = (xc * xc).mean(-1, keepdim=True)
    rs = 1.0 / torch.sqrt(var + eps)
    zz = xc * rs
    e_mu = K * x.abs().mean(-1, keepdim=True) + U * mu.abs()
    e_rs = 0.5 * ((K + 4 * U) + e_mu ** 2 * rs ** 2) + 3 * U  # relative
    e_z = rs * (e_mu + U * xc.abs()) + zz.abs() * (e_rs + 2 * U)
    gain, offset = gain.double(), offset.double()
    y = zz * gain + offset
    out = {"y": y, "e_y": e_z * gain.abs() + 3 * U * ((zz * gain).abs() + offset.abs())}
    if dy is None:
        return out
    dy = dy.double()
    d = dy * gain
    m1 = d.mean(-1, keepdim=True)
    m2 = (d * zz).mean(-1, keepdim=True)
    out["dx"] = rs * (d - m1 - zz * m2)
    e_m1 = K * d.abs().mean(-1, keepdim=True)
    e_m2 = K * (d * zz).abs().mean(-1, keepdim=True) + (d.abs() * e_z).mean(-1, keepdim=True)
    size = d.abs() + m1.abs() + (zz * m2).abs()
    out["e_dx"] = rs * (5 * U * size + e_m1 + zz.abs() * e_m2 + e_z * m2.abs()) + out["dx"].abs() * (e_rs + 2 * U)
    out["pz"], out["p1"] = dy * zz, dy
    out["e_pz"] = dy.abs() * e_z + 2 * U * (dy * zz).abs()
    return out


def sum_bound(p, e_p, rows):
    """Error bound of a float32 sum over ``rows`` (dim -2) of terms p, each off by e_p: at most
    ceil(rows / 32) + 32 + 64 additions follow one another (rows of a team, teams, joined partials)."""
    return e_p.sum(-2) + (rows / 32 + 97) * U * p.abs().sum(-2)


def assert_within(got, want, bound, dtype, what=""):
    """|got - want| <= bound + one rounding to dtype, elementwise."""
    got, want = got.double().cpu(), want.double().cpu()
    bound = bound.double().cpu()
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # rounding of subnormals
    limit = bound + half_step(dtype) * (want.abs() + bound) + tiny
    bad = ~((got - want).abs() <= limit)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, worst "
                           f"{float(((got - want).abs() / limit)[bad].max()):.3g} times the limit")


# ---------------------------------------------------------------------------- predictor block
def modulate(x, shift, scale):
    return x * (1 + scale) + shift


class Attention(torch.nn.Module):
    def __init__(self, dim, heads, dim_head):
        super().__init__()
        self.heads = heads
        self.norm = torch.nn.LayerNorm(dim)
        self.to_qkv = torch.nn.Linear(dim, 3 * heads * dim_head, bias=False)
        self.to_out = torch.nn.Sequential(torch.nn.Linear(heads * dim_head, dim))

    def forward(self, x):
        b, t, _ = x.shape
        q, k, v = (u.view(b, t, self.heads, -1).transpose(1, 2) for u in self.to_qkv(self.norm(x)).chunk(3, -1))
        s = q @ k.transpose(-1, -2) / math.sqrt(q.shape[-1])
        s = s.masked_fill(torch.ones(t, t, dtype=torch.bool, device=x.device).triu(1), -math.inf)
        return self.to_out((s.softmax(-1) @ v).transpose(1, 2).reshape(b, t, -1))


class ConditionalBlock(torch.nn.Module):
    def __init__(self, dim, heads, dim_head, mlp_dim):
        super().__init__()
        self.attn = Attention(dim, heads, dim_head)
        self.mlp = torch.nn.Sequential(torch.nn.LayerNorm(dim), torch.nn.Linear(dim, mlp_dim), torch.nn.GELU(),
                                       torch.nn.Linear(mlp_dim, dim))
        self.norm1 = torch.nn.LayerNorm(dim, elementwise_affine=False, eps=1e-6)
        self.norm2 = torch.nn.LayerNorm(dim, elementwise_affine=False, eps=1e-6)
        self.adaLN_modulation = torch.nn.Sequential(torch.nn.SiLU(), torch.nn.Linear(dim, 6 * dim))

    def forward(self, x, c):
        sa, ka, ga, sm, km, gm = self.adaLN_modulation(c).chunk(6, dim=-1)
        x = x + ga * self.attn(modulate(self.norm1(x), sa, ka))
        return x + gm * self.mlp(modulate(self.norm2(x), sm, km))


class TinyPredictor(torch.nn.Module):
    def __init__(self, dim=64, depth=2, heads=2, dim_head=32, mlp_dim=128):
        super().__init__()
        self.layers = torch.nn.ModuleList(ConditionalBlock(dim, heads, dim_head, mlp_dim) for _ in range(depth))
        self.norm = torch.nn.LayerNorm(dim)

    def forward(self, x, c):
        for block in self.layers:
            x = block(x, c)
        return self.norm(x)
