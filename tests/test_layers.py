"""Layer operators (smrt_amd.autoencode.layers) without a GPU: what they refuse, and the C entries' own argument checks."""
import ctypes as C

import pytest
import torch

from smrt_amd import _hip
from smrt_amd.autoencode import (PackedRows, dense, dense_backward, dense_grouped, dense_grouped_backward, layer_norm,
                                 layer_norm_backward, pack_rows, unpack_rows)


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def packed(rows, cols, dtype=torch.float32):
    b = -(-cols // 32)
    return PackedRows(t(rows, 32 * b, dtype=torch.int8), t(rows, b, dtype=torch.uint8), cols, dtype)


REFUSED = [
    ("x is no tensor", TypeError, lambda: dense([[1.0]], t(1, 1))),
    ("x of another type", ValueError, lambda: dense(t(2, 3, dtype=torch.float64), t(3, 4, dtype=torch.float64))),
    ("x 1-d", ValueError, lambda: dense(t(3), t(3, 4))),
    ("x 3-d", ValueError, lambda: dense(t(2, 2, 3), t(3, 4))),
    ("weight of another type", ValueError, lambda: dense(t(2, 3), t(3, 4, dtype=torch.bfloat16))),
    ("weight of another depth", ValueError, lambda: dense(t(2, 3), t(4, 4))),
    ("weight transposed", ValueError, lambda: dense(t(2, 3), t(4, 3).t())),
    ("rows that overlap", ValueError, lambda: dense(t(1, 3).expand(2, 3), t(3, 4))),
    ("bias shape", ValueError, lambda: dense(t(2, 3), t(3, 4), t(3))),
    ("bias 2-d", ValueError, lambda: dense(t(2, 3), t(3, 4), t(1, 4))),
    ("residual shape", ValueError, lambda: dense(t(2, 3), t(3, 4), residual=t(1, 4))),
    ("residual type", ValueError, lambda: dense(t(2, 3), t(3, 4), residual=t(2, 4, dtype=torch.float16))),
    ("out shape", ValueError, lambda: dense(t(2, 3), t(3, 4), out=t(2, 5))),
    ("activation", ValueError, lambda: dense(t(2, 3), t(3, 4), activation="gelu")),
    ("activation no text", ValueError, lambda: dense(t(2, 3), t(3, 4), activation=[])),
    ("save", ValueError, lambda: dense(t(2, 3), t(3, 4), save="all")),
    ("requires grad", ValueError, lambda: dense(t(2, 3).requires_grad_(), t(3, 4))),
    ("packed x in the forward pass", TypeError, lambda: dense(packed(2, 3), t(3, 4))),
    ("backward without saved", ValueError, lambda: dense_backward(t(2, 4), t(2, 3), t(3, 4), activation="relu")),
    ("backward grad shape", ValueError, lambda: dense_backward(t(2, 5), t(2, 3), t(3, 4))),
    ("backward x rows", ValueError, lambda: dense_backward(t(2, 4), t(3, 3), t(3, 4))),
    ("backward packed of another type", ValueError, lambda: dense_backward(t(2, 4), packed(2, 3, torch.float16), t(3, 4))),
    ("backward packed of another shape", ValueError, lambda: dense_backward(t(2, 4), packed(2, 4), t(3, 4))),
    ("ends missing", TypeError, lambda: dense_grouped(t(2, 3), None, t(1, 3, 4))),
    ("ends int32", ValueError, lambda: dense_grouped(t(2, 3), t(1, dtype=torch.int32), t(1, 3, 4))),
    ("ends length", ValueError, lambda: dense_grouped(t(2, 3), t(2, dtype=torch.int64), t(1, 3, 4))),
    ("no groups", ValueError, lambda: dense_grouped(t(2, 3), t(0, dtype=torch.int64), t(0, 3, 4))),
    ("grouped weight 2-d", ValueError, lambda: dense_grouped(t(2, 3), t(1, dtype=torch.int64), t(3, 4))),
    ("grouped weights that overlap", ValueError, lambda: dense_grouped(t(2, 3), t(2, dtype=torch.int64), t(1, 3, 4).expand(2, 3, 4))),
    ("grouped bias 1-d", ValueError, lambda: dense_grouped(t(2, 3), t(2, dtype=torch.int64), t(2, 3, 4), t(4))),
    ("grouped backward ends", ValueError, lambda: dense_grouped_backward(t(2, 4), t(2, 3), t(3, dtype=torch.int64), t(2, 3, 4))),
    ("norm no columns", ValueError, lambda: layer_norm(t(2, 0))),
    ("norm too wide", ValueError, lambda: layer_norm(t(1, 32769))),
    ("norm eps", ValueError, lambda: layer_norm(t(2, 3), eps=-1.0)),
    ("norm eps nan", ValueError, lambda: layer_norm(t(2, 3), eps=float("nan"))),
    ("norm bias alone", ValueError, lambda: layer_norm(t(2, 3), None, t(3))),
    ("norm weight type", ValueError, lambda: layer_norm(t(2, 3), t(3, dtype=torch.bfloat16))),
    ("norm bias type", ValueError, lambda: layer_norm(t(2, 3, dtype=torch.bfloat16), t(3), t(3, dtype=torch.bfloat16))),
    ("norm weight length", ValueError, lambda: layer_norm(t(2, 3), t(4))),
    ("norm backward mean", ValueError, lambda: layer_norm_backward(t(2, 3), t(2, 3), t(3), t(2))),
    ("norm backward rstd type", ValueError, lambda: layer_norm_backward(t(2, 3), t(2, 3), t(2), t(2, dtype=torch.float16))),
    ("pack int", ValueError, lambda: pack_rows(t(2, 3, dtype=torch.int8))),
    ("unpack tensor", TypeError, lambda: unpack_rows(t(2, 3))),
    ("packed q shape", ValueError, lambda: PackedRows(t(2, 3, dtype=torch.int8), t(2, 1, dtype=torch.uint8), 3, torch.float32)),
    ("packed scale shape", ValueError, lambda: PackedRows(t(2, 64, dtype=torch.int8), t(2, 1, dtype=torch.uint8), 33, torch.float32)),
    ("packed dtype", ValueError, lambda: PackedRows(t(2, 32, dtype=torch.int8), t(2, 1, dtype=torch.uint8), 3, torch.float64)),
]


@pytest.mark.parametrize("what,error,call", REFUSED, ids=[r[0] for r in REFUSED])
def test_refused(what, error, call):
    with pytest.raises(error):
        call()


@pytest.mark.parametrize("call", [
    lambda: dense(t(2, 3), t(3, 4)), lambda: dense_backward(t(2, 4), t(2, 3), t(3, 4)),
    lambda: dense_grouped(t(2, 3), t(1, dtype=torch.int64), t(1, 3, 4)),
    lambda: layer_norm(t(2, 3)), lambda: layer_norm_backward(t(2, 3), t(2, 3), t(2), t(2)),
    lambda: pack_rows(t(2, 3)), lambda: unpack_rows(packed(2, 3))])
def test_no_cpu_fallback(call):
    with pytest.raises(_hip.HipLibraryError):
        call()


def _dense_args(**kw):
    """A sound call on made-up addresses that is refused for what `kw` changes; nothing is launched before the checks."""
    base = dict(dtype=0, activation=3, rows=4, k=8, n=16, groups=1, x=0x10000, ldx=8, w=0x20000, ldw=16, w_stride=0, bias_stride=16,
                y=0x30000, ldy=16, a=0x40000, lda=16, grad=0x50000, ldg=16, dx=0x60000, lddx=8, dw=0x70000, lddw=16, dw_stride=128, db=0x80000)
    return _hip.Dense(**{**base, **kw})


FORWARD_BAD = [dict(dtype=3), dict(dtype=-1), dict(activation=5), dict(rows=-1), dict(rows=1 << 31), dict(k=1 << 31), dict(groups=0),
               dict(groups=2), dict(groups=1 << 16, ends=0x1000), dict(ldx=7), dict(ldx=(1 << 21) + 1), dict(ldw=(1 << 21) + 1), dict(ldw=15), dict(ldy=15), dict(lda=15), dict(x=0), dict(w=0), dict(y=0),
               dict(x_scale=0x90000), dict(residual=0x100000, ldr=15), dict(groups=2, ends=0x1000, w_stride=64), dict(w_stride=-1),
               dict(groups=2, ends=0x1000, w_stride=128, bias=0x1000, bias_stride=15),
               dict(a_scale=0x90000, lda=16), dict(a_scale=0x90000, lda=32, ld_a_scale=0),
               dict(y=0x10000), dict(y=0x20010), dict(residual=0x30010, ldr=16), dict(residual=0x30000, ldr=20)]


@pytest.mark.parametrize("kw", FORWARD_BAD, ids=str)
def test_dense_forward_entry_refuses(kw):
    args = _dense_args(**kw)
    assert _hip.load().smrt_dense_forward(C.byref(args), None) == -1
    assert b"smrt_dense_forward" in _hip.load().smrt_last_error()


BACKWARD_BAD = [dict(dtype=3), dict(groups=0), dict(ldg=15), dict(lddx=7), dict(lddw=15), dict(grad=0), dict(a=0), dict(lda=15), dict(x=0),
                dict(x_scale=0x90000, ldx=8), dict(x_scale=0x90000, ldx=32, ld_x_scale=0), dict(a_scale=0x90000, lda=16),
                dict(groups=2, ends=0x1000, w_stride=128, dw_stride=100)]


@pytest.mark.parametrize("kw", BACKWARD_BAD, ids=str)
def test_dense_backward_entry_refuses(kw):
    args = _dense_args(**kw)
    assert _hip.load().smrt_dense_backward(C.byref(args), 0xa0000, 1 << 20, None) == -1


def test_entries_refuse_null_and_small_workspaces():
    lib = _hip.load()
    assert lib.smrt_dense_forward(None, None) == -1
    assert lib.smrt_dense_backward(None, None, 0, None) == -1
    assert lib.smrt_dense_backward_workspace(None) == -1
    assert lib.smrt_layer_norm_forward(None, None) == -1
    assert lib.smrt_layer_norm_backward(None, None, 0, None) == -1
    assert lib.smrt_layer_norm_backward_workspace(None) == -1
    args = _dense_args()
    assert lib.smrt_dense_backward_workspace(C.byref(args)) == 0          # a few rows have all their gradients from one launch
    args = _dense_args(rows=300)
    need = lib.smrt_dense_backward_workspace(C.byref(args))
    assert need > 0
    assert lib.smrt_dense_backward(C.byref(args), 0xa0000, need - 1, None) == -1
    assert lib.smrt_dense_backward(C.byref(args), None, need, None) == -1
    norm = dict(dtype=1, rows=4000, n=64, eps=1e-5, x=0x10000, ldx=64, y=0x200000, ldy=64, mean=0x900000, rstd=0xa00000, grad=0xb00000, ldg=64,
                dx=0xc00000, lddx=64, dw=0xd00000, db=0xe00000)
    args = _hip.LayerNorm(**norm)
    need = lib.smrt_layer_norm_backward_workspace(C.byref(args))
    assert need > 0
    assert lib.smrt_layer_norm_backward(C.byref(args), 0x10000, need - 1, None) == -1
    for kw in (dict(dtype=9), dict(n=0), dict(n=32769), dict(rows=-1), dict(ldx=63), dict(ldy=63), dict(x=0), dict(y=0), dict(mean=0), dict(eps=-1.0),
               dict(x_scale=0x1000), dict(y=0x10080)):
        args = _hip.LayerNorm(**{**norm, **kw})
        assert lib.smrt_layer_norm_forward(C.byref(args), None) == -1, kw
    for kw in (dict(ldg=63), dict(lddx=63), dict(grad=0), dict(x_scale=0x1000, ld_x_scale=1)):
        args = _hip.LayerNorm(**{**norm, **kw})
        assert lib.smrt_layer_norm_backward(C.byref(args), 0x10000, 1 << 30, None) == -1, kw


def test_pack_entries_refuse():
    lib = _hip.load()
    good = [0, 0x1000, 40, 4, 40, 0x2000, 64, 0x3000, 2]
    for i, v in ((0, 3), (1, 0), (2, 39), (3, -1), (4, -1), (5, 0), (6, 63), (7, 0), (8, 1)):
        bad = list(good)
        bad[i] = v
        assert lib.smrt_pack_rows(*bad, None) == -1, (i, v)
        dt, x, ldx, rows, n, q, ldq, s, lds = bad
        assert lib.smrt_unpack_rows(dt, q, ldq, s, lds, rows, n, x, ldx, None) == -1, (i, v)


def test_entries_refuse_shared_memory():
    lib = _hip.load()
    for kw in (dict(a=0x30010), dict(a=0x10000), dict(a=0x20020), dict(residual=0x40000, ldr=16), dict(a_scale=0x30000, lda=32, ld_a_scale=1)):
        args = _dense_args(**kw)
        assert lib.smrt_dense_forward(C.byref(args), None) == -1 and b"overlaps" in lib.smrt_last_error(), kw
    for kw in (dict(dx=0x50000), dict(dx=0x10000), dict(dx=0x40000), dict(dw=0x20000), dict(dw=0x60000), dict(db=0x70000), dict(db=0x50000)):
        args = _dense_args(**kw)
        assert lib.smrt_dense_backward(C.byref(args), 0xa0000, 1 << 20, None) == -1 and b"overlaps" in lib.smrt_last_error(), kw
    args = _dense_args(rows=300)
    assert lib.smrt_dense_backward(C.byref(args), 0x50000, 1 << 20, None) == -1 and b"overlaps" in lib.smrt_last_error()
    norm = dict(dtype=1, rows=4000, n=64, eps=1e-5, x=0x10000, ldx=64, weight=0x100000, y=0x200000, ldy=64, mean=0x900000, rstd=0xa00000, grad=0xb00000,
                ldg=64, dx=0xc00000, lddx=64, dw=0xd00000, db=0xe00000)
    for kw in (dict(y=0x100000), dict(mean=0x200010), dict(rstd=0x900000)):
        args = _hip.LayerNorm(**{**norm, **kw})
        assert lib.smrt_layer_norm_forward(C.byref(args), None) == -1 and b"overlaps" in lib.smrt_last_error(), kw
    for kw in (dict(dx=0xb00000), dict(dx=0x10000), dict(dw=0x100000), dict(db=0xd00000), dict(db=0x900000)):
        args = _hip.LayerNorm(**{**norm, **kw})
        assert lib.smrt_layer_norm_backward(C.byref(args), 0x2000000, 1 << 30, None) == -1 and b"overlaps" in lib.smrt_last_error(), kw
    assert lib.smrt_pack_rows(0, 0x1000, 40, 4, 40, 0x1000, 64, 0x3000, 2, None) == -1
    assert lib.smrt_unpack_rows(0, 0x2000, 64, 0x1010, 2, 4, 40, 0x1000, 40, None) == -1


def test_class_decoders_refuse():
    from sklearn.exceptions import NotFittedError
    from smrt_amd.autoencode import ClassDecoders, VariationalAutoEncoder
    with pytest.raises(ValueError):
        ClassDecoders([])
    with pytest.raises(ValueError):
        ClassDecoders([VariationalAutoEncoder(4, 2)], dtype=torch.float64)
    with pytest.raises(NotFittedError):
        ClassDecoders([VariationalAutoEncoder(4, 2)])


def test_the_package_is_imported_without_torch():
    """Only the layers need torch; asking for one of their names brings it in."""
    import os
    import subprocess
    import sys
    code = """
import sys
import smrt_amd.autoencode as a, smrt_amd.balance, smrt_amd.utils
assert "torch" not in sys.modules
names = ["ClassDecoders", "PackedRows", "class_decoders", "dense", "dense_backward", "dense_grouped", "dense_grouped_backward", "layer_norm",
         "layer_norm_backward", "layers", "pack_rows", "unpack_rows"]
assert set(names) <= set(a.__all__) and set(names) <= set(dir(a)) and "torch" not in sys.modules
assert a.dense is a.layers.dense and a.ClassDecoders is a.class_decoders.ClassDecoders and "torch" in sys.modules
assert sorted(set(a.layers.__all__ + a.class_decoders.__all__ + ["layers", "class_decoders"])) == sorted(names)
try:
    a.no_such_name
except AttributeError as e:
    assert "no_such_name" in str(e)
else:
    raise AssertionError
from smrt_amd.autoencode import *
assert layer_norm is a.layer_norm and VariationalAutoEncoder is a.VariationalAutoEncoder
"""
    subprocess.run([sys.executable, "-c", code], check=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def test_entries_refuse_outputs_over_any_input():
    """Biases, ends, scale bytes and a norm's input count as much as the matrices do."""
    lib = _hip.load()

    def refused(fn, args, *rest):
        assert fn(C.byref(args), *rest, None) == -1 and b"overlaps" in lib.smrt_last_error(), args
    groups = dict(rows=40, groups=2, ends=0x200000, w_stride=128)
    for kw in (dict(bias=0x30010), dict(bias=0x40010), dict(bias=0x2fffc), dict(bias=0x30000, residual=0x30000, ldr=16),
               dict(groups, bias=0x30100, bias_stride=16), dict(groups, bias=0x2ff80, bias_stride=40), dict(groups, ends=0x30010), dict(groups, ends=0x2fff8),
               dict(groups, ends=0x3fff8), dict(rows=4, ends=0x30000),
               dict(a_scale=0x90000, lda=32, ld_a_scale=1, bias=0x8fff0), dict(a_scale=0x90000, lda=32, ld_a_scale=1, residual=0x90000, ldr=16),
               dict(groups, a_scale=0x90000, lda=32, ld_a_scale=1, ends=0x8fff8)):
        refused(lib.smrt_dense_forward, _dense_args(**kw))
    packed_x, packed_a = dict(x_scale=0x90000, ldx=32, ld_x_scale=1), dict(a_scale=0x98000, lda=32, ld_a_scale=1)
    for kw in (dict(groups, dx=0x200008), dict(groups, db=0x1ffffc), dict(groups, dw=0x1fff00), dict(rows=4, ends=0x60000),
               dict(packed_x, dx=0x90000), dict(packed_x, dw=0x8ff00), dict(packed_x, db=0x90000), dict(packed_a, dx=0x98000), dict(packed_a, db=0x97ffc),
               dict(packed_x, db=0x10008)):
        refused(lib.smrt_dense_backward, _dense_args(**kw), 0xa0000, 1 << 20)
    refused(lib.smrt_dense_backward, _dense_args(rows=300, a_scale=0xa0010, lda=32, ld_a_scale=1), 0xa0000, 1 << 20)
    refused(lib.smrt_dense_backward, _dense_args(rows=300, groups=2, ends=0xa0100, w_stride=128), 0xa0000, 1 << 20)
    norm = dict(dtype=1, rows=4000, n=64, eps=1e-5, x=0x10000, ldx=64, weight=0x100000, y=0x200000, ldy=64, mean=0x900000, rstd=0xa00000, grad=0xb00000,
                ldg=64, dx=0xc00000, lddx=64, dw=0xd00000, db=0xe00000)
    for kw in (dict(mean=0x10000), dict(rstd=0x12000), dict(y=0x10000, mean=0x10000)):
        refused(lib.smrt_layer_norm_forward, _hip.LayerNorm(**{**norm, **kw}))
    for kw in (dict(x_scale=0xd00000, ld_x_scale=2), dict(x_scale=0xcffff0, ld_x_scale=2, dx=None), dict(x=0xd00000 - 3999 * 96 - 48, ldx=96, n=40, x_scale=0x80000, ld_x_scale=2)):
        refused(lib.smrt_layer_norm_backward, _hip.LayerNorm(**{**norm, **kw}), 0x2000000, 1 << 30)


def test_tangents_are_refused():
    """A dual tensor's tangent would be lost without a word.  Tensors without one are taken as ever, integers among them."""
    from torch.autograd import forward_ad
    cases = [(lambda d: dense(d(2, 3), t(3, 4))), (lambda d: dense(t(2, 3), d(3, 4))), (lambda d: dense(t(2, 3), t(3, 4), d(4))),
             (lambda d: dense(t(2, 3), t(3, 4), residual=d(2, 4))), (lambda d: dense(t(2, 3), t(3, 4), out=d(2, 4))),
             (lambda d: dense_backward(d(2, 4), t(2, 3), t(3, 4))), (lambda d: dense_backward(t(2, 4), d(2, 3), t(3, 4))),
             (lambda d: dense_backward(t(2, 4), t(2, 3), t(3, 4), d(2, 4), activation="tanh")),
             (lambda d: dense_grouped(t(2, 3), t(2, dtype=torch.int64), d(2, 3, 4))), (lambda d: dense_grouped(t(2, 3), t(2, dtype=torch.int64), t(2, 3, 4), d(2, 4))),
             (lambda d: layer_norm(d(2, 3))), (lambda d: layer_norm(t(2, 3), d(3))), (lambda d: layer_norm(t(2, 3), t(3), d(3))),
             (lambda d: layer_norm_backward(d(2, 3), t(2, 3), t(2), t(2))), (lambda d: layer_norm_backward(t(2, 3), t(2, 3), d(2), t(2))), (lambda d: pack_rows(d(2, 3)))]
    with forward_ad.dual_level():
        for call in cases:
            with pytest.raises(ValueError, match="tangent"):
                call(lambda *s: forward_ad.make_dual(t(*s), t(*s)))
            with pytest.raises(_hip.HipLibraryError):                # past all checks of the arguments
                call(t)
        with pytest.raises(_hip.HipLibraryError):
            dense_backward(t(2, 4), packed(2, 3), t(3, 4))
