"""What is timed of the training operators: layer norm, adaptive layer norm, gradient clipping.

Fine-tuning the world model that the planner plans with runs, per step, a LayerNorm or an
AdaLN-modulated LayerNorm at every sub-layer (forward and backward) and one global-norm clip
over all gradients. A case is a dict of plain values; ``prepare`` makes its tensors on the GPU,
``run`` makes one pass and returns every output, ``exact`` gives the same outputs in 64 bits.

With ``own`` false a pass is elementary torch operations in float32; with ``own`` true it is
the calls a user makes of ``lewm_flash_b200``.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MAX_ELEMENTS = 1 << 28            # elements of the largest activation or gradient set
MAX_ACTIVATION_BYTES = 1 << 29    # bytes of the largest activation

# Predictor parameter shapes at width 192 / 6 layers / 16 heads of 64 / MLP 768 / 3 frames
# (the package's default model description, in state-dict order).
PREDICTOR = (
    [(1, 3, 192)]
    + 6 * [(1152, 192), (1152,), (192,), (192,), (3 * 1024, 192), (192, 1024), (192,), (192,), (192,),
           (768, 192), (768,), (192, 768), (192,)]
    + [(192,), (192,), (10, 10, 1), (10,), (768, 10), (768,), (192, 768), (192,)]
)


def listed():
    """The timed cases."""
    return [
        # ---- layer norm: (rows, width), row-wise over the width
        # One candidate's window of three tokens at the predictor's width, inference: latency.
        {"name": "ln_window_forward", "op": "ln", "train": False, "rows": 3, "width": 192, "dtype": "f32",
         "ptype": "f32", "affine": "both", "pad": 0},
        # The encoder's tokens: 64 images of 257 tokens at width 192, bf16 activations, f32 weights.
        {"name": "ln_encoder_tokens", "op": "ln", "train": True, "rows": 64 * 257, "width": 192, "dtype": "bf16",
         "ptype": "f32", "affine": "both", "pad": 0},
        # Odd width and row count, rows cut out of a wider buffer: nothing is 16-byte aligned.
        {"name": "ln_odd_strided", "op": "ln", "train": True, "rows": 8191, "width": 1011, "dtype": "f16",
         "ptype": "f16", "affine": "weight", "pad": 6},
        # The projector head's hidden width (2048) over a large batch of tokens.
        {"name": "ln_projector_large", "op": "ln", "train": True, "rows": 131072, "width": 2048, "dtype": "bf16",
         "ptype": "f32", "affine": "both", "pad": 0},
        # ---- adaptive layer norm: (batch, tokens, width), modulation per token or per sequence
        # One planner call's windows, per-token modulation chunked out of the AdaLN Linear's output.
        {"name": "ada_window_train", "op": "ada", "train": True, "batch": 300, "tokens": 3, "width": 192,
         "dtype": "f32", "ctype": "f32", "per_token": True, "chunks": 6},
        # 64 environments of 300 candidates, inference under bf16.
        {"name": "ada_windows_forward", "op": "ada", "train": False, "batch": 64 * 300, "tokens": 3, "width": 192,
         "dtype": "bf16", "ctype": "bf16", "per_token": True, "chunks": 6},
        # One modulation row per image for its 257 tokens, at the wider predictor's width.
        {"name": "ada_sequence_train", "op": "ada", "train": True, "batch": 64, "tokens": 257, "width": 384,
         "dtype": "bf16", "ctype": "f32", "per_token": False, "chunks": 6},
        # Long sequences with one modulation row each, float32 training at a large width.
        {"name": "ada_long_train", "op": "ada", "train": True, "batch": 9, "tokens": 8209, "width": 1536,
         "dtype": "f32", "ctype": "f32", "per_token": False, "chunks": 2},
        # ---- global gradient norm and clipping
        # The gradient of 30 refined action sequences: one small tensor, latency.
        {"name": "clip_actions", "op": "clip", "shapes": "actions", "dtype": "f32", "norm": "2", "fraction": 0.1, "align": 64},
        # All gradients of the default predictor, float32 (they fit the L2 cache).
        {"name": "clip_predictor", "op": "clip", "shapes": "predictor", "dtype": "f32", "norm": "2",
         "fraction": 0.3, "align": 64},
        # Many tensors of odd sizes, half of them bf16 and half float32, packed back to back in
        # flat buffers (so most start at unaligned addresses).
        {"name": "clip_ragged_mixed", "op": "clip", "shapes": "drawn", "count": 523, "total": 33554467,
         "dtype": "mixed", "norm": "2", "fraction": 0.7, "align": 1},
        # A large bf16 model's gradients, far beyond the L2 cache.
        {"name": "clip_large", "op": "clip", "shapes": "drawn", "count": 291, "total": MAX_ELEMENTS,
         "dtype": "bf16", "norm": "2", "fraction": 0.3, "align": 64},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges."""
    op = rng.choice(["ln", "ada", "clip"])
    if op == "clip":
        total = _log_int(rng, 1, MAX_ELEMENTS)
        dtype = rng.choice(["f32", "bf16", "f16", "mixed"])
        if dtype in ("f32", "mixed"):
            total = min(total, MAX_ELEMENTS // 2)
        return {"op": "clip", "shapes": "drawn", "count": min(total, _log_int(rng, 1, 1500)), "total": total,
                "dtype": dtype, "norm": rng.choice(["2", "2", "inf"]), "fraction": 10.0 ** rng.uniform(-1.5, 0.5),
                "align": rng.choice([1, 64, 64])}
    dtype = rng.choice(["f32", "bf16", "f16"])
    size = DTYPES[dtype].itemsize
    cap = min(MAX_ELEMENTS, MAX_ACTIVATION_BYTES // size)
    width = _log_int(rng, 1, 8192)
    if rng.random() < 0.5:
        width = max(8, width // 8 * 8)
    ptype = rng.choice(["f32", dtype])
    train = rng.random() < 0.75
    rows = min(_log_int(rng, 1, 131072), max(1, cap // (width + 8)))
    if op == "ln":
        return {"op": "ln", "train": train, "rows": rows, "width": width, "dtype": dtype, "ptype": ptype,
                "affine": rng.choice(["both", "both", "weight", "none"]), "pad": rng.choice([0, 0, 0, 5, 8])}
    tokens = min(rows, _log_int(rng, 1, 16384))
    return {"op": "ada", "train": train, "batch": max(1, rows // tokens), "tokens": tokens, "width": width,
            "dtype": dtype, "ctype": ptype, "per_token": rng.random() < 0.5 and rows * width * 3 <= cap,
            "chunks": rng.choice([2, 3, 6])}


# ---------------------------------------------------------------------------- inputs
def _shapes(case):
    """(shape, dtype) of every gradient of a clip case."""
    if case["shapes"] == "actions":
        shapes = [(1, 30, 5, 10)]
    elif case["shapes"] == "predictor":
        shapes = PREDICTOR
    else:
        # Parameter sizes spread over their logarithm, as biases and matrices are, summing to total.
        count, total = case["count"], case["total"]
        r = random.Random(1000003 * count + total)
        w = [math.exp(r.uniform(0.0, 9.0)) for _ in range(count)]
        free = total - count
        sizes = [1 + int(free * v / sum(w)) for v in w]
        sizes[0] += total - sum(sizes)
        shapes = [(n,) for n in sizes]
    kinds = ["bf16", "f32"] if case["dtype"] == "mixed" else [case["dtype"]]
    return [(s, DTYPES[kinds[i % len(kinds)]]) for i, s in enumerate(shapes)]


def _scales(case):
    """Standard deviation of each gradient: four decades apart; float16 ones are loss-scaled."""
    top = 2 if case["dtype"] == "f16" else -1
    return [10.0 ** (top - i % 4) for i in range(len(_shapes(case)))]


def _max_norm(case):
    """The clipping threshold: a fraction of the norm that the gradients are drawn with."""
    scales = _scales(case)
    if case["norm"] == "inf":
        return case["fraction"] * 4.0 * max(scales)
    return case["fraction"] * math.sqrt(sum(math.prod(s) * v * v for (s, _), v in zip(_shapes(case), scales)))


def _activation(g, rows, width, dtype, buffer_width=None):
    """Residual-stream-like rows: a scale and an offset per row, some loud channels, and a zero
    row (padding) in every 61."""
    x = torch.randn(rows, buffer_width or width, device="cuda", generator=g)
    x *= torch.rand(rows, 1, device="cuda", generator=g).mul_(1.5).add_(0.25)
    x += torch.randn(rows, 1, device="cuda", generator=g)
    x[:, :: 97] *= 6.0
    x[60::61] = 0.0
    return x.to(dtype)


def prepare(case, seed):
    """The tensors of a case, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "clip":
        # Gradients live in one flat buffer per type, each starting at a multiple of `align`
        # elements (what lies between them is zero); so does what the pass writes.
        shapes, align, length, places = _shapes(case), case["align"], {}, []
        for shape, dtype in shapes:
            places.append(length.get(dtype, 0))
            length[dtype] = places[-1] + (math.prod(shape) + align - 1) // align * align
        flat = {d: torch.zeros(n, device="cuda", dtype=d) for d, n in length.items()}
        out = {d: torch.zeros_like(t) for d, t in flat.items()}
        views = [[buf[d][at:at + math.prod(s)].view(s) for (s, d), at in zip(shapes, places)] for buf in (flat, out)]
        for t, scale in zip(views[0], _scales(case)):
            t.copy_(randn(*t.shape).mul_(scale))
        return {"case": case, "flat": flat, "grads": views[0], "out_flat": out, "out": views[1],
                "max_norm": _max_norm(case)}
    dtype = DTYPES[case["dtype"]]
    width, train = case["width"], case["train"]
    if case["op"] == "ln":
        rows, ptype = case["rows"], DTYPES[case["ptype"]]
        x = _activation(g, rows, width, dtype, width + case["pad"])[:, :width]
        weight = (1.0 + 0.1 * randn(width)).to(ptype) if case["affine"] != "none" else None
        bias = (0.1 * randn(width)).to(ptype) if case["affine"] == "both" else None
        state = {"case": case, "x": x, "weight": weight, "bias": bias}
        leaves = [x, weight, bias]
        shape = (rows, width)
    else:
        batch, tokens, ctype = case["batch"], case["tokens"], DTYPES[case["ctype"]]
        x = _activation(g, batch * tokens, width, dtype).view(batch, tokens, width)
        mod = (0.3 * randn(batch, tokens if case["per_token"] else 1, case["chunks"] * width)).to(ctype)
        shift, scale = mod.chunk(case["chunks"], dim=-1)[:2]
        state = {"case": case, "x": x, "shift": shift, "scale": scale}
        leaves = [x, shift, scale]
        shape = (batch, tokens, width)
    if train:
        state["dy"] = randn(*shape).mul_(0.05).to(dtype)
        for t in leaves:
            if t is not None:
                t.requires_grad_(True)
    return state


# ---------------------------------------------------------------------------- one pass
EPS = {"ln": 1e-5, "ada": 1e-6}


def run(state):
    """One pass: (y, gradients...) of a norm, or the clipped gradients and their norm."""
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import lewm_flash_b200 as lf

    case = state["case"]
    if case["op"] == "clip":
        _, norm = lf.clip_grads(state["grads"], state["max_norm"], norm_type=float(case["norm"]), out=state["out"])
        return [norm, *state["out_flat"].values()]
    x = state["x"]
    if case["op"] == "ln":
        leaves = [t for t in (x, state["weight"], state["bias"]) if t is not None]
        y = lf.layer_norm(x, state["weight"], state["bias"], eps=EPS["ln"])
    else:
        leaves = [x, state["shift"], state["scale"]]
        y = lf.ada_layer_norm(x, state["shift"], state["scale"], eps=EPS["ada"])
    if not case["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, leaves, state["dy"])]


@torch.no_grad()
def _run_plain(state):
    case = state["case"]
    if case["op"] == "clip":
        grads = state["grads"]
        if case["norm"] == "inf":
            norm = torch.stack([t.float().abs().max() for t in grads]).max()
        else:
            norm = torch.stack([(t.float() * t.float()).sum(dtype=torch.float64) for t in grads]).sum().sqrt().float()
        coef = torch.clamp(state["max_norm"] / (norm + 1e-6), max=1.0)
        for t, out in zip(grads, state["out"]):
            out.copy_(t.float() * coef)
        return [norm, *state["out_flat"].values()]
    x = state["x"].float()
    xc = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + EPS[case["op"]])
    xhat = xc * rstd
    if case["op"] == "ln":
        w = None if state["weight"] is None else state["weight"].float()
        b = None if state["bias"] is None else state["bias"].float()
    else:
        w, b = 1.0 + state["scale"].float(), state["shift"].float()
    y = xhat if w is None else xhat * w
    if b is not None:
        y = y + b
    out = [y.to(state["x"].dtype)]
    if not case["train"]:
        return out
    dy = state["dy"].float()
    d = dy if w is None else dy * w
    dx = rstd * (d - d.mean(-1, keepdim=True) - xhat * (d * xhat).mean(-1, keepdim=True))
    out.append(dx.to(state["x"].dtype))
    if case["op"] == "ln":
        if w is not None:
            out.append((dy * xhat).sum(0).to(state["weight"].dtype))
        if b is not None:
            out.append(dy.sum(0).to(state["bias"].dtype))
        return out
    dshift, dscale = dy, dy * xhat
    if not case["per_token"]:
        dshift, dscale = dshift.sum(1, keepdim=True), dscale.sum(1, keepdim=True)
    return out + [dshift.to(state["shift"].dtype), dscale.to(state["scale"].dtype)]


# ---------------------------------------------------------------------------- 64 bits
@torch.no_grad()
def exact(case, seed):
    """The outputs of ``run`` from the definitions in float64."""
    state = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "clip":
        if case["norm"] == "inf":
            norm = max(float(t.abs().max()) for t in state["grads"])
        else:
            norm = math.sqrt(sum(float(torch.square(t.to(f64)).sum()) for t in state["grads"]))
        coef = min(1.0, state["max_norm"] / (norm + 1e-6))
        return [torch.tensor(norm, dtype=f64)] + [t.to(f64) * coef for t in state["flat"].values()]
    n = case["width"]
    x = state["x"].detach().to(f64)
    var, mu = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    sigma = torch.sqrt(var + EPS[case["op"]])
    z = (x - mu) / sigma
    del x
    if case["op"] == "ln":
        gain = torch.ones(n, dtype=f64, device=z.device) if state["weight"] is None else state["weight"].to(f64)
        offset = torch.zeros(n, dtype=f64, device=z.device) if state["bias"] is None else state["bias"].to(f64)
    else:
        gain, offset = state["scale"].to(f64) + 1.0, state["shift"].to(f64)
    out = [z * gain + offset]
    if not case["train"]:
        return out
    # d/dx of z: (I - 1 1^T / n - z z^T / n) / sigma, applied to the gradient at z.
    dy = state["dy"].to(f64)
    dz = dy * gain
    along_one = dz.sum(-1, keepdim=True) / n
    along_z = (dz * z).sum(-1, keepdim=True) / n
    out.append((dz - along_one - z * along_z) / sigma)
    del dz
    if case["op"] == "ln":
        if state["weight"] is not None:
            out.append(torch.einsum("rc,rc->c", dy, z))
        if state["bias"] is not None:
            out.append(torch.einsum("rc->c", dy))
    elif case["per_token"]:
        out += [dy, dy * z]
    else:
        out += [torch.einsum("btc->bc", dy).unsqueeze(1), torch.einsum("btc,btc->bc", dy, z).unsqueeze(1)]
    return out


# ---------------------------------------------------------------------------- cost
def work(case):
    """Bytes and operations a pass cannot do without: every input read once, every output
    written once."""
    if case["op"] == "clip":
        n = total = 0
        for shape, dtype in _shapes(case):
            k = math.prod(shape)
            n += k
            total += k * dtype.itemsize
        return {"bytes": 2 * total + 4, "flops": 3 * n}
    size = DTYPES[case["dtype"]].itemsize
    width = case["width"]
    if case["op"] == "ln":
        rows = case["rows"]
        params = {"both": 2, "weight": 1, "none": 0}[case["affine"]] * width * DTYPES[case["ptype"]].itemsize
    else:
        rows = case["batch"] * case["tokens"]
        mods = rows if case["per_token"] else case["batch"]
        params = 2 * mods * width * DTYPES[case["ctype"]].itemsize
    n = rows * width
    # Forward: x in, y out; training: dy in, dx out, and the gradients of the parameters
    # (of the scale only of those per token: d shift is dy itself, yet it is an output too).
    passes = 4 if case["train"] else 2
    return {"bytes": passes * n * size + (2 if case["train"] else 1) * params, "flops": (22 if case["train"] else 8) * n}
