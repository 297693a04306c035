"""Training operators, no GPU: argument checks of the Python functions and of the C ABI, row
strides, overlap detection, and which modules install_training_norms routes."""

import ctypes as C
import math

import numpy as np
import pytest
import torch

import lewm_flash_b200 as lf
from lewm_flash_b200 import _lib, training
from tests.training_reference import ConditionalBlock, TinyPredictor

z = torch.zeros


@pytest.mark.parametrize("call,msg", [
    (lambda: lf.layer_norm(z(())), "last dim"),
    (lambda: lf.layer_norm(z(3, 0)), "last dim"),
    (lambda: lf.layer_norm(z(3, 8, dtype=torch.float64)), "float32, bfloat16 or float16"),
    (lambda: lf.layer_norm(z(3, 8, dtype=torch.int32)), "float32, bfloat16 or float16"),
    (lambda: lf.layer_norm(z(3, 8).to_sparse()), "dense"),
    (lambda: lf.layer_norm(torch._neg_view(z(3, 8))), "negated"),
    (lambda: lf.grad_norm([torch._neg_view(z(3))]), "negated"),
    (lambda: lf.layer_norm(z(3, 8), z(7)), r"weight must be \(8,\)"),
    (lambda: lf.layer_norm(z(3, 8), z(8), z(1, 8)), r"bias must be \(8,\)"),
    (lambda: lf.layer_norm(z(3, 8), z(8), z(8).half()), "one type"),
    (lambda: lf.layer_norm(z(3, 8), eps=-1.0), "eps"),
    (lambda: lf.layer_norm(z(3, 8), eps=math.nan), "eps"),
    (lambda: lf.layer_norm(z(3, 8), z(8), z(8)), "need a CUDA device"),
    (lambda: lf.ada_layer_norm(z(2, 3, 8), z(2, 3, 8), z(2, 1, 8)), "one shape and type"),
    (lambda: lf.ada_layer_norm(z(2, 3, 8), z(2, 1, 8), z(2, 1, 8).half()), "one shape and type"),
    (lambda: lf.ada_layer_norm(z(2, 3, 8), z(3, 8), z(3, 8)), "do not modulate"),
    (lambda: lf.ada_layer_norm(z(2, 3, 8), z(1, 3, 8), z(1, 3, 8)), "do not modulate"),
    (lambda: lf.ada_layer_norm(z(2, 3, 8), z(2, 1, 1), z(2, 1, 1)), "do not modulate"),
    (lambda: lf.ada_layer_norm(z(2, 3, 8), z(2, 2, 3, 8), z(2, 2, 3, 8)), "do not modulate"),
    (lambda: lf.ada_layer_norm(z(2, 3, 8), z(()), z(())), "do not modulate"),
    (lambda: lf.ada_layer_norm(z(2, 3, 8), z(2, 1, 8), z(2, 1, 8)), "need a CUDA device"),
    (lambda: lf.grad_norm([z(3)], 1.0), "norm_type must be 2 or inf"),
    (lambda: lf.grad_norm([z(3, dtype=torch.float64)]), "float32, bfloat16 or float16"),
    (lambda: lf.grad_norm([z(3)]), "need a CUDA device"),
    (lambda: lf.grad_norm([z(3), z(3, device="meta")]), "one device per call"),
    (lambda: lf.clip_grads([z(3)], -1.0), "max_norm must be >= 0"),
    (lambda: lf.clip_grads([z(3)], math.nan), "max_norm must be >= 0"),
    (lambda: lf.clip_grads([z(3)], 1.0, out=[]), "out has 0 tensors"),
    (lambda: lf.clip_grads([z(3)], 1.0, out=[z(4)]), r"out\[0\] must be"),
    (lambda: lf.clip_grads([z(3)], 1.0, out=[z(3).half()]), r"out\[0\] must be"),
    (lambda: lf.clip_grads([z(3)], 1.0, out=[z(6)[::2]]), "contiguous"),
    (lambda: lf.clip_grads([z(3)], 1.0), "need a CUDA device"),
])
def test_refused_arguments(call, msg):
    with pytest.raises(ValueError, match=msg):
        call()


def test_non_tensors_are_type_errors():
    with pytest.raises(TypeError):
        lf.layer_norm(np.zeros((3, 8)))
    with pytest.raises(TypeError):
        lf.grad_norm([z(3), 4.0])


def test_overlapping_gradients_are_refused():
    g = z(8)
    with pytest.raises(ValueError, match="overlap"):
        lf.clip_grads([g, g], 1.0, out=[g, g])
    with pytest.raises(ValueError, match="overlap"):
        lf.clip_grads([g[:5], g[3:]], 1.0, out=[g[:5], g[3:]])
    with pytest.raises(ValueError, match="overlap"):  # an output on another gradient
        lf.clip_grads([g[:4], g[4:]], 1.0, out=[g[4:], z(4)])
    p = torch.nn.Parameter(z(3))
    p.grad = z(3)
    with pytest.raises(ValueError, match="overlap"):
        lf.clip_grad_norm_([p, p], 1.0)
    p.grad = z(1).expand(3)
    with pytest.raises(ValueError, match="shares memory"):
        lf.clip_grad_norm_([p], 1.0)


def test_overlap_rule():
    def overlap(src, dst, size):
        return training._ops().overlap(src, dst, size)

    assert not overlap([16, 32], [16, 32], [16, 16])    # in place, back to back
    assert not overlap([16, 16], [32, 48], [16, 16])    # one source read twice
    assert not overlap([0, 64], [64 * 4, 64 * 8], [64, 64])
    assert not overlap([5, 5, 9], [5, 5, 9], [0, 0, 4])  # empty tensors meet nothing
    assert overlap([16, 16], [16, 16], [4, 4])          # the same one twice, in place
    assert overlap([0, 64], [128, 130], [4, 4])         # outputs meet
    assert overlap([0, 64], [2, 128], [4, 4])           # an output on its own source, shifted
    assert overlap([0, 64], [64, 128], [4, 4])          # an output on another source
    assert overlap([0, 64, 0], [0, 64, 128], [4, 4, 4])  # a source read while it is clipped in place


def test_empty_gradient_lists():
    assert lf.grad_norm([]).item() == 0.0
    out, norm = lf.clip_grads([], 1.0)
    assert out == [] and norm.item() == 0.0
    assert lf.clip_grad_norm_([torch.nn.Parameter(z(2))], 1.0).item() == 0.0


@pytest.mark.parametrize("make,copied,stride", [
    (lambda: z(4, 5, 8), False, 8),
    (lambda: z(4, 5, 24)[..., 8:16], False, 24),
    (lambda: z(4, 5, 8)[:, :1], False, 40),
    (lambda: z(4, 5, 8)[:, :3], True, 8),
    (lambda: z(5, 4, 8).transpose(0, 1), True, 8),
    (lambda: z(1, 8).expand(6, 8), False, 0),
    (lambda: z(8).expand(3, 4, 8), False, 0),
    (lambda: z(8, 4).t(), True, 8),
    (lambda: z(6, 2)[:, :1], False, 2),
    (lambda: z(3, 1, 7, 8)[:, :, ::7], False, 56),
    (lambda: z(0, 8), False, 8),
])
def test_rows_are_read_in_place_where_they_step_evenly(make, copied, stride):
    t = make()
    rows, step = training._ops().rows(t)
    assert (rows is not t) == copied and step == stride
    n = t.shape[-1]
    if t.numel():
        flat = torch.arange(0, t.untyped_storage().nbytes() // 4, dtype=torch.float32)
        t.untyped_storage().copy_(flat.untyped_storage())
        rows, step = training._ops().rows(t)
        got = torch.as_strided(rows, (t.numel() // n, n), (step, 1 if n > 1 else 1), rows.storage_offset())
        assert torch.equal(got, t.reshape(-1, n))


# ---------------------------------------------------------------------------- C ABI
def desc(rows=4, width=8, x_stride=8, group=0, a_stride=0, b_stride=0, x_type=0, p_type=0, eps=1e-5):
    return _lib.NormDescC(rows, width, x_stride, group, a_stride, b_stride, x_type, p_type, eps)


BUF = (C.c_float * 64)()
P = C.addressof(BUF)


@pytest.mark.parametrize("kw,status,msg", [
    (dict(rows=-1), 1, "rows"), (dict(width=0), 1, "width"), (dict(width=(1 << 24) + 1), 2, "width"),
    (dict(x_type=3), 1, "element type"), (dict(p_type=-1), 1, "element type"), (dict(eps=-1.0), 1, "eps"),
    (dict(eps=math.nan), 1, "eps"), (dict(x_stride=-8), 1, "stride"), (dict(group=3), 1, "whole groups"),
    (dict(group=-1), 1, "whole groups"), (dict(group=2, a_stride=-1), 1, "stride"),
])
def test_c_abi_norm_refusals(kw, status, msg):
    lib = _lib.lib()
    d = desc(**kw)
    assert lib.lewm_norm_forward(C.byref(d), P, None, None, P, None, 0, None) == status
    assert msg in lib.lewm_last_error(None).decode()
    assert lib.lewm_norm_backward(C.byref(d), P, 8, P, None, P, P, None, None, None, 0, 0, None) == status
    assert lib.lewm_norm_workspace(C.byref(d)) == 0


def test_c_abi_norm_null_pointers_and_workspace():
    lib = _lib.lib()
    assert lib.lewm_norm_forward(None, P, None, None, P, None, 0, None) == 1
    d = desc()
    assert lib.lewm_norm_forward(C.byref(d), None, None, None, P, None, 0, None) == 1
    assert lib.lewm_norm_forward(C.byref(d), P, None, None, None, None, 0, None) == 1
    a = desc(group=2, a_stride=8, b_stride=8)
    assert lib.lewm_norm_forward(C.byref(a), P, None, P, P, None, 0, None) == 1  # no scale
    assert lib.lewm_norm_backward(C.byref(d), P, 8, P, None, None, P, None, None, None, 0, 0, None) == 1  # no stats
    assert lib.lewm_norm_backward(C.byref(d), P, -1, P, None, P, P, None, None, None, 0, 0, None) == 1
    big = desc(rows=4096)
    need = lib.lewm_norm_workspace(C.byref(big))
    assert need > 0 and need % (2 * 8 * 4) == 0
    assert lib.lewm_norm_backward(C.byref(big), P, 8, P, P, P, P, P, None, P, need - 1, 0, None) == 1
    assert "workspace" in lib.lewm_last_error(None).decode()
    assert lib.lewm_norm_backward(C.byref(big), P, 8, P, P, P, P, P, None, P // 16 * 16 + 8, need, 0, None) == 1
    assert "aligned" in lib.lewm_last_error(None).decode()
    # Pointers off their elements.
    for args in ((P + 2, None, None, P, None), (P, P + 2, None, P, None), (P, None, None, P + 1, None),
                 (P, None, None, P, P + 2)):
        assert lib.lewm_norm_forward(C.byref(d), *args, 0, None) == 1
        assert "not aligned to its element" in lib.lewm_last_error(None).decode()
    for args in ((P + 2, 8, P, None, P, P, None, None), (P, 8, P + 2, None, P, P, None, None),
                 (P, 8, P, None, P, P + 2, None, None), (P, 8, P, None, P + 2, P, None, None),
                 (P, 8, P, None, P, P, P + 2, None), (P, 8, P, None, P, P, None, P + 1)):
        assert lib.lewm_norm_backward(C.byref(d), *args, None, 0, 0, None) == 1
    # Nothing to do: no rows, or no gradient asked for.
    e = desc(rows=0)
    assert lib.lewm_norm_forward(C.byref(e), None, None, None, None, None, 0, None) == 0
    assert lib.lewm_norm_backward(C.byref(d), None, 8, None, None, None, None, None, None, None, 0, 0, None) == 0
    assert lib.lewm_norm_backward(C.byref(e), P, 8, P, None, P, None, P, None, None, 0, 0, None) == 1
    assert "no rows" in lib.lewm_last_error(None).decode()


@pytest.mark.parametrize("width", [1, 64, 65, 192, 512, 1011, 2048, 16384, 16385, 100003])
@pytest.mark.parametrize("rows,group", [(1, 0), (7, 0), (4097, 0), (1 << 33, 0), (900, 1), (1 << 20, 3), (64 * 257, 257),
                                        (2, 1), (1 << 33, 1 << 31)])
def test_workspace_holds_whole_partial_sums(width, rows, group):
    d = desc(rows=rows, width=width, x_stride=width, group=group, a_stride=width, b_stride=width)
    need = _lib.lib().lewm_norm_workspace(C.byref(d))
    assert need % (2 * width * 4) == 0
    groups = rows // group if group else 1
    assert need == 0 or need // (2 * width * 4) >= 2 * groups  # a group alone needs none
    # Partial sums never outgrow what the GPU keeps in flight by much.
    assert need // (2 * width * 4) <= max(2 * groups, groups + 148 * 64)


def test_c_abi_gradient_refusals():
    lib = _lib.lib()
    src = (C.c_void_p * 2)(P, P + 64)
    counts = (C.c_int64 * 2)(8, 8)
    types = (C.c_int32 * 2)(0, 0)

    def norm(src=src, counts=counts, types=types, n=2, kind=0, ws=P, out=P):
        return lib.lewm_grad_norm(src, counts, types, n, kind, ws, out, 0, None)

    assert norm(n=-1) == 1 and norm(kind=2) == 1 and norm(ws=None) == 1 and norm(out=None) == 1
    assert norm(src=None) == 1 and norm(counts=None) == 1 and norm(types=None) == 1
    assert norm(ws=(P + 15) // 16 * 16 + 4) == 1
    assert norm(types=(C.c_int32 * 2)(0, 3)) == 1 and norm(counts=(C.c_int64 * 2)(8, -1)) == 1
    assert norm(src=(C.c_void_p * 2)(P, None)) == 1 and norm(src=(C.c_void_p * 2)(P, P + 66)) == 1
    assert norm(n=(1 << 20) + 1) == 2

    def clip(dst=src, max_norm=1.0, norm_in=None, n=2):
        return lib.lewm_grad_clip(src, dst, counts, types, n, 0, max_norm, norm_in, P, P + 128, 0, None)

    assert clip(dst=None) == 1 and clip(max_norm=-1.0) == 1 and clip(max_norm=math.nan) == 1
    assert clip(norm_in=P + 128) == 1 and clip(dst=(C.c_void_p * 2)(P, None)) == 1


# ---------------------------------------------------------------------------- module routing
def test_install_routes_norms_and_blocks_and_removes_them():
    model = TinyPredictor(dim=16, depth=2, heads=2, dim_head=8, mlp_dim=32)
    x, c = torch.randn(2, 3, 16), torch.randn(2, 3, 16)
    want = model(x, c)
    keys = list(model.state_dict())
    handle = lf.install_training_norms(model)
    blocks = [n for n, m in model.named_modules() if isinstance(m, ConditionalBlock)]
    norms = [n for n, m in model.named_modules() if isinstance(m, torch.nn.LayerNorm)]
    assert sorted(handle.modules) == sorted(blocks + norms) and len(blocks) == 2
    assert list(model.state_dict()) == keys
    with pytest.raises(ValueError, match="need a CUDA device"):
        model(x, c)
    assert lf.install_training_norms(model).modules == []  # nothing is routed twice
    handle.remove()
    assert torch.equal(model(x, c), want)


def test_install_leaves_other_modules_alone():
    class Scaled(torch.nn.LayerNorm):
        def forward(self, x):
            return 2 * super().forward(x)

    class Renamed(torch.nn.LayerNorm):
        pass

    class Block(ConditionalBlock):  # could do anything with its parts
        pass

    model = torch.nn.Sequential(torch.nn.LayerNorm((3, 8)), torch.nn.Linear(8, 8), torch.nn.BatchNorm1d(8),
                                torch.nn.LayerNorm(8), Scaled(8), Renamed(8), Block(8, 1, 8, 8))
    assert lf.install_training_norms(model).modules == ["3", "5", "6.attn.norm", "6.mlp.0", "6.norm1", "6.norm2"]


@pytest.mark.parametrize("value", [0.0, -1.0, math.nan])
def test_cem_gd_gradient_clip_must_be_positive(value):
    with pytest.raises(ValueError, match="gd_max_grad_norm must be positive"):
        lf.B200CEMGDSolver(model=None, gd_max_grad_norm=value)
    assert lf.B200CEMGDSolver(model=None).gd_max_grad_norm is None


def test_header_sizes_have_no_second_copy():
    """LEWM_GRAD_WORKSPACE stands in the header alone, where the extension takes it from: a copy in the
    binding would go stale unnoticed, as lewm_grad_* cannot check what it is given."""
    header = _lib.PKG.parent / "include" / "lewm_b200.h"
    assert "#define LEWM_GRAD_WORKSPACE 32768" in header.read_text()
    assert not [n for n in vars(_lib) if "WORKSPACE" in n]
