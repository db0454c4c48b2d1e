"""Layers on device tensors: the dense layer, layer norm and the 8-bit form of activations, each with its gradients.

A ``VariationalAutoEncoder`` or ``AutoEncoder`` trains and runs a whole net behind one handle.  These are the layers by
themselves, for nets that are put together from them: a deeper classifier on a balanced set, residual blocks between an
encoder's layers, several classes' decoders over one batch.  In the reference a layer exists only inside its TensorFlow
graph (smrt/autoencode/layer.py:348-464).

    y = act(x W + b) + r        dense, dense_backward                    (activations and weight layout as in the estimators)
    the same, a weight a class  dense_grouped, dense_grouped_backward    (rows sorted by class)
    y = layer norm of x         layer_norm, layer_norm_backward
    activations in 8 bits       pack_rows, unpack_rows, PackedRows       (what the backward calls take in a tensor's place)

Tensors are ``float32``, ``bfloat16`` or ``float16`` on one GPU, 2-d, with a row's elements next to each other and rows at
any distance (up to 2^21 elements for what a product reads); sums are fp32.  Work is queued on the device's current torch stream and nothing waits for it, so the calls
can be captured into graphs.  They take no part in torch's autograd -- the gradients are calls of their own -- and
refuse a tensor that requires grad while grad mode is on, or that has a tangent.  There is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version      # a tensor of the caller's that is written over: autograd may have kept it

from .. import _hip

__all__ = ["dense", "dense_backward", "dense_grouped", "dense_grouped_backward", "layer_norm", "layer_norm_backward",
           "pack_rows", "unpack_rows", "PackedRows"]

_Tensor = torch.Tensor
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_BLOCK = 32                                      # columns that share a scale byte


# A small layer is over in a few microseconds, so the checks have a short way for the usual argument -- a plain tensor of the
# right type, device and layout, outside of every level of forward-mode differentiation (number -1) -- and words only for the others.
def _tensor(t, name, dim, dtype, dev):
    """Checks any tensor argument; ``dtype`` None: one of the three types, ``dev`` None: any device."""
    if type(t) is _Tensor and t.dtype is dtype and t.get_device() == dev and not t.requires_grad and t.is_contiguous() and t.dim() == dim \
            and forward_ad._current_level < 0:
        return t
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor, got %s" % (name, type(t).__name__))
    if t.dim() != dim:
        raise ValueError("%s must have %d dimension(s), got shape %r" % (name, dim, tuple(t.shape)))
    if dtype is None:
        if t.dtype not in _DTYPES:
            raise ValueError("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
    elif t.dtype != dtype:
        raise ValueError("%s must be %s, got %s" % (name, dtype, t.dtype))
    if dev is not None and t.get_device() != dev:
        raise ValueError("%s is on %s, expected %s" % (name, t.device, "the CPU" if dev < 0 else "cuda:%d" % dev))
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s requires grad, and the layer calls take no part in autograd: detach it, or call under torch.no_grad()" % name)
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError("%s has a tangent, and the layer calls take no part in autograd: hand over its primal part" % name)
    if t.shape[-1] > 1 and t.stride(-1) != 1 and t.numel():
        raise ValueError("the elements of a row of %s must lie next to each other (strides %r)" % (name, t.stride()))
    return t


def _ld(t, name):
    """Leading dimension of a matrix (of the last two dimensions)."""
    rows, cols = t.shape[-2:]
    if rows <= 1 or cols == 0:
        return max(cols, 1)
    ld = t.stride(-2)
    if ld < cols:
        raise ValueError("the rows of %s overlap (strides %r)" % (name, t.stride()))
    return ld


def _matrix(t, name, dtype, dev):
    """Checks a matrix argument: ``(rows, cols, leading dimension)``."""
    if type(t) is _Tensor and (t.dtype is dtype or dtype is None and t.dtype in _DTYPES) and t.get_device() == dev and not t.requires_grad \
            and forward_ad._current_level < 0:
        stride = t.stride()
        if len(stride) == 2 and stride[1] == 1:
            rows, cols = t.shape
            if stride[0] >= cols > 0:
                return rows, cols, stride[0] if rows > 1 else cols          # a single row has no distance to another
    _tensor(t, name, 2, dtype, dev)
    return t.shape[0], t.shape[1], _ld(t, name)


def _shape(t, name, shape):
    if t.shape != shape:
        raise ValueError("%s must have shape %r, got %r" % (name, shape, tuple(t.shape)))


def _device_of(t, name):
    """Ordinal of a tensor's GPU, -1 for the CPU."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor, got %s" % (name, type(t).__name__))
    return t.get_device()


def _on_gpu(dev):
    if dev < 0:
        raise _hip.HipLibraryError("the layer calls run on an MI355X; there is no CPU fallback (got tensors on the CPU)")


# what torch.cuda.current_stream(dev).cuda_stream and torch.cuda.current_device() come to, without their objects
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _call(dev, fn, *args):
    """``fn(*args, stream)`` on the device's current stream, with that device current."""
    if _current_device() == dev:
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        raise _hip.HipLibraryError("%s failed (%d): %s" % (fn.__name__, rc, _hip.load().smrt_last_error().decode()))


def _activation(name):
    try:
        return _hip.ACTIVATION_IDS[name]
    except (KeyError, TypeError):
        raise ValueError("activation must be one of %r, got %r" % (sorted(_hip.ACTIVATION_IDS), name)) from None


# ------------------------------------------------------------------------------------------------ 8-bit form
class PackedRows(object):
    """A matrix of activations held in 8 bits: what a backward pass reads in place of the tensor it was made from.

    ``q`` int8 ``[rows, cols rounded up to 32]``, ``scale`` uint8 ``[rows, cols / 32]``: 32 columns of a row share a power of two,
    a value is ``q * 2 ** (scale - 127)`` with ``|q| <= 127`` -- off by at most 1/126 of the block's largest magnitude (half a step of
    ``q``, of which that magnitude takes 63.5 or more).  The two ends of the scales differ: at the lowest (1; 103 in float16) a value is off by half of its step, 2^-127
    (0 in float16, whose numbers are whole steps there), which takes the smallest ones to zero; at the highest (249; 137 in float16), where 64 steps would be an infinity,
    ``|q| <= 63`` and a value is off by up to 1/64.  A block that held an infinity or a NaN stands for 32 NaNs (scale 255).
    ``dtype`` is the type of the values."""

    __slots__ = ("q", "scale", "cols", "dtype")

    def __init__(self, q, scale, cols, dtype):
        cols = int(cols)
        if dtype not in _DTYPES:
            raise ValueError("dtype must be float32, bfloat16 or float16, got %s" % dtype)
        dev = _device_of(q, "q")
        _tensor(q, "q", 2, torch.int8, dev)
        _tensor(scale, "scale", 2, torch.uint8, dev)
        blocks = -(-cols // _BLOCK)
        _shape(q, "q", (q.shape[0], blocks * _BLOCK))
        _shape(scale, "scale", (q.shape[0], blocks))
        _ld(q, "q"), _ld(scale, "scale")
        self.q, self.scale, self.cols, self.dtype = q, scale, cols, dtype

    @property
    def shape(self):
        return (self.q.shape[0], self.cols)

    @property
    def device(self):
        return self.q.device

    def __repr__(self):
        return "PackedRows(shape=%r, dtype=%s, device=%s)" % (self.shape, self.dtype, self.q.device)


def _new_packed(rows, cols, dtype, device):
    blocks = -(-cols // _BLOCK)
    p = object.__new__(PackedRows)
    p.q = torch.empty((rows, blocks * _BLOCK), dtype=torch.int8, device=device)
    p.scale = torch.empty((rows, blocks), dtype=torch.uint8, device=device)
    p.cols, p.dtype = cols, dtype
    return p


def pack_rows(x):
    """The 8-bit form of ``x`` ``[rows, cols]`` (``PackedRows``)."""
    dev = _device_of(x, "x")
    rows, cols, ld = _matrix(x, "x", None, dev)
    _on_gpu(dev)
    p = _new_packed(rows, cols, x.dtype, x.device)
    _call(dev, _hip.load().smrt_pack_rows, _DTYPES[x.dtype], x.data_ptr(), ld, rows, cols, p.q.data_ptr(), p.q.shape[1], p.scale.data_ptr(),
          p.scale.shape[1])
    return p


def unpack_rows(packed):
    """The values that ``packed`` stands for, a tensor ``[rows, cols]`` of ``packed.dtype``."""
    if not isinstance(packed, PackedRows):
        raise TypeError("packed must be PackedRows, got %s" % type(packed).__name__)
    q, scale, cols = packed.q, packed.scale, packed.cols
    dev, rows = q.get_device(), q.shape[0]
    _on_gpu(dev)
    out = torch.empty((rows, cols), dtype=packed.dtype, device=q.device)
    _call(dev, _hip.load().smrt_unpack_rows, _DTYPES[packed.dtype], q.data_ptr(), _ld(q, "q"), scale.data_ptr(), _ld(scale, "scale"), rows, cols,
          out.data_ptr(), cols or 1)
    return out


def _kept(t, name, rows, cols, dtype, dev):
    """A tensor or PackedRows of an earlier pass: ``(pointer, ld, scale pointer, scale ld)``."""
    if isinstance(t, PackedRows):
        q, scale = t.q, t.scale
        if t.dtype != dtype or q.shape[0] != rows or t.cols != cols or q.get_device() != dev:
            raise ValueError("%s must be a %s matrix of shape %r on the others' device, got %r" % (name, dtype, (rows, cols), t))
        return q.data_ptr(), _ld(q, name), scale.data_ptr(), _ld(scale, name)
    r, c, ld = _matrix(t, name, dtype, dev)
    if r != rows or c != cols:
        _shape(t, name, (rows, cols))
    return t.data_ptr(), ld, None, 0


# ------------------------------------------------------------------------------------------------ dense
def _weights(weight, bias, dtype, dev, ends):
    """Checks of a weight ``[k, n]`` or ``[groups, k, n]``, its bias and the groups' ends: ``(k, n, groups, ldw, w_stride, bias pointer, bias_stride)``."""
    if ends is None:
        k, n, ldw = _matrix(weight, "weight", dtype, dev)
        if bias is None:
            return k, n, 1, ldw, 0, None, n
        _tensor(bias, "bias", 1, dtype, dev)
        if bias.shape[0] != n:
            _shape(bias, "bias", (n,))
        return k, n, 1, ldw, 0, bias.data_ptr(), n
    _tensor(weight, "weight", 3, dtype, dev)
    groups, k, n = weight.shape
    _tensor(ends, "ends", 1, torch.int64, dev)
    _shape(ends, "ends", (groups,))
    if not 1 <= groups <= 65535:
        raise ValueError("between 1 and 65535 groups are supported, got %d" % groups)
    ldw, w_stride = _ld(weight, "weight"), weight.stride(0) if groups > 1 else 0
    if groups > 1 and w_stride < (k - 1) * ldw + n:
        raise ValueError("the weights of the groups overlap (strides %r)" % (weight.stride(),))
    if bias is None:
        return k, n, groups, ldw, w_stride, None, n
    b_rows, b_cols, bias_stride = _matrix(bias, "bias", dtype, dev)
    if b_rows != groups or b_cols != n:
        _shape(bias, "bias", (groups, n))
    return k, n, groups, ldw, w_stride, bias.data_ptr(), bias_stride


def _dense(x, ends, weight, bias, residual, activation, save, out):
    act = _activation(activation)
    if save is not None and save not in ("activation", "packed"):
        raise ValueError("save must be None, 'activation' or 'packed', got %r" % (save,))
    dev = _device_of(x, "x")
    rows, xk, ldx = _matrix(x, "x", None, dev)
    dtype = x.dtype
    k, n, groups, ldw, w_stride, b_ptr, bias_stride = _weights(weight, bias, dtype, dev, ends)
    if xk != k:
        raise ValueError("x has %d columns, weight has shape %r" % (xk, tuple(weight.shape)))
    r_ptr, ldr = None, 0
    if residual is not None:
        r_rows, r_cols, ldr = _matrix(residual, "residual", dtype, dev)
        if r_rows != rows or r_cols != n:
            _shape(residual, "residual", (rows, n))
        r_ptr = residual.data_ptr()
    if out is None:
        _on_gpu(dev)
        y, ldy = x.new_empty((rows, n)), n or 1
    else:
        y_rows, y_cols, ldy = _matrix(out, "out", dtype, dev)
        if y_rows != rows or y_cols != n:
            _shape(out, "out", (rows, n))
        _on_gpu(dev)
        increment_version(out)
        y = out
    saved, a_ptr, lda, s_ptr, lds = None, None, 0, None, 0
    if save is not None and act != 1:                      # the identity's derivative needs nothing
        if save == "packed":
            saved = _new_packed(rows, n, dtype, x.device)
            a_ptr, lda, s_ptr, lds = saved.q.data_ptr(), saved.q.shape[1], saved.scale.data_ptr(), saved.scale.shape[1]
        elif residual is None:
            saved = y
        else:
            saved = x.new_empty((rows, n))
            a_ptr, lda = saved.data_ptr(), n
    args = _hip.Dense(_DTYPES[dtype], act, rows, k, n, groups, out is not None, None if ends is None else ends.data_ptr(),
                      x.data_ptr(), ldx, None, 0, weight.data_ptr(), ldw, w_stride, b_ptr, bias_stride, r_ptr, ldr, y.data_ptr(), ldy,
                      a_ptr, lda, s_ptr, lds)
    _call(dev, _hip.load().smrt_dense_forward, C.byref(args))
    return y if save is None else (y, saved)


def _dense_backward(grad, x, ends, weight, saved, activation, need_x, need_weight, need_bias):
    act = _activation(activation)
    dev = _device_of(grad, "grad")
    rows, gn, ldg = _matrix(grad, "grad", None, dev)
    dtype, device = grad.dtype, grad.device
    k, n, groups, ldw, w_stride, _, _ = _weights(weight, None, dtype, dev, ends)
    if gn != n:
        raise ValueError("grad has %d columns, weight has shape %r" % (gn, tuple(weight.shape)))
    x_ptr, ldx, xs_ptr, ld_xs = _kept(x, "x", rows, k, dtype, dev)
    a_ptr, lda, as_ptr, ld_as = None, 0, None, 0
    if act != 1:
        if saved is None:
            raise ValueError("the gradient of %r needs what the forward pass saved" % activation)
        a_ptr, lda, as_ptr, ld_as = _kept(saved, "saved", rows, n, dtype, dev)
    _on_gpu(dev)
    dx = grad.new_empty((rows, k)) if need_x else None
    dw = grad.new_empty(weight.shape) if need_weight else None
    db = grad.new_empty((n,) if ends is None else (groups, n)) if need_bias else None
    args = _hip.Dense(_DTYPES[dtype], act, rows, k, n, groups, 0, None if ends is None else ends.data_ptr(),
                      x_ptr, ldx, xs_ptr, ld_xs, weight.data_ptr(), ldw, w_stride, None, n, None, 0, None, 0, a_ptr, lda, as_ptr, ld_as,
                      grad.data_ptr(), ldg, dx.data_ptr() if need_x else None, k or 1, dw.data_ptr() if need_weight else None, n or 1, k * n,
                      db.data_ptr() if need_bias else None)
    lib, ref = _hip.load(), C.byref(args)
    size = lib.smrt_dense_backward_workspace(ref)
    work = torch.empty((size,), dtype=torch.uint8, device=device) if size > 0 else None
    _call(dev, lib.smrt_dense_backward, ref, None if work is None else work.data_ptr(), size)
    return dx, dw, db


def dense(x, weight, bias=None, residual=None, activation="identity", save=None, out=None):
    """``act(x @ weight + bias) + residual`` in one launch: ``x`` ``[rows, k]``, ``weight`` ``[k, n]`` (the estimators' layout).

    ``save`` keeps what ``dense_backward`` needs, and makes the result ``(y, saved)``: ``"activation"`` the activation's value (``y`` itself
    without a residual), ``"packed"`` its 8-bit form, written by the same launch.  For the identity, whose derivative needs
    nothing, ``saved`` is None.  ``out`` receives ``y``; it may be the residual itself, and no other input."""
    return _dense(x, None, weight, bias, residual, activation, save, out)


def dense_backward(grad, x, weight, saved=None, activation="identity", need_x=True, need_weight=True, need_bias=True):
    """Gradients ``(dx, dweight, dbias)`` of ``dense`` from ``grad`` = d loss / d y (None where not needed; the residual's gradient is ``grad``).

    ``x`` and ``saved`` are the forward pass's tensors, or their 8-bit forms: the gradients are then those at the values the 8 bits
    stand for.

    In a 16-bit type ``dz = grad * act'`` is rounded once to that type before it is multiplied into ``dx`` and ``dweight``, as an operand of the matrix cores; ``dbias`` is
    summed from the values before.  Kernels for a few rows (at most 256) multiply ``dz`` in fp32."""
    return _dense_backward(grad, x, None, weight, saved, activation, need_x, need_weight, need_bias)


def dense_grouped(x, ends, weight, bias=None, residual=None, activation="identity", save=None, out=None):
    """``dense`` with a weight for each class: rows ``[ends[g-1], ends[g])`` of ``x`` are multiplied by ``weight[g]`` (``[groups, k, n]``,
    bias ``[groups, n]``), all classes in one launch.  ``ends`` is an int64 tensor on the device, the running sum of the classes' row counts;
    classes may be empty.  An end below the one before it or past the rows counts as that bound.  Rows behind the last end are zero in a result
    made here, and left as they were in ``out``."""
    return _dense(x, _ends(ends), weight, bias, residual, activation, save, out)


def dense_grouped_backward(grad, x, ends, weight, saved=None, activation="identity", need_x=True, need_weight=True, need_bias=True):
    """Gradients ``(dx [rows, k], dweight [groups, k, n], dbias [groups, n])`` of ``dense_grouped``; zero for a class without rows, and
    for rows that are in no class.  ``dz`` is rounded as in ``dense_backward``."""
    return _dense_backward(grad, x, _ends(ends), weight, saved, activation, need_x, need_weight, need_bias)


def _ends(ends):
    if ends is None:
        raise TypeError("ends must be a torch tensor, got NoneType")
    return ends


# ------------------------------------------------------------------------------------------------ layer norm
def _norm_weight(weight, bias, dtype, dev, n):
    """``(weight is float32, weight pointer, bias pointer)``"""
    if weight is None:
        if bias is not None:
            raise ValueError("bias without weight is not supported")
        return 0, None, None
    if not isinstance(weight, torch.Tensor) or weight.dtype not in (dtype, torch.float32):
        raise ValueError("weight must be a tensor of %s or float32" % dtype)
    _tensor(weight, "weight", 1, weight.dtype, dev)
    if weight.shape[0] != n:
        _shape(weight, "weight", (n,))
    if bias is not None:
        _tensor(bias, "bias", 1, weight.dtype, dev)
        if bias.shape[0] != n:
            _shape(bias, "bias", (n,))
    return weight.dtype is torch.float32, weight.data_ptr(), None if bias is None else bias.data_ptr()


def layer_norm(x, weight=None, bias=None, eps=1e-5, out=None):
    """``(y, mean, rstd)``: each row of ``x`` ``[rows, n]`` less its mean, over ``sqrt(variance + eps)``, times ``weight`` plus ``bias``
    (``[n]``, of ``x``'s type or float32).  ``mean`` and ``rstd`` are float32 ``[rows]``, for the backward pass.  1 <= n <= 32768.
    ``out`` receives ``y`` and may be ``x``."""
    dev = _device_of(x, "x")
    rows, n, ldx = _matrix(x, "x", None, dev)
    dtype, device = x.dtype, x.device
    if not 1 <= n <= 32768:
        raise ValueError("layer norm takes 1 to 32768 columns, got %d" % n)
    if not eps >= 0.0:
        raise ValueError("eps must be >= 0, got %r" % (eps,))
    w_f32, w_ptr, b_ptr = _norm_weight(weight, bias, dtype, dev, n)
    if out is None:
        _on_gpu(dev)
        y, ldy = x.new_empty((rows, n)), n
    else:
        y_rows, y_cols, ldy = _matrix(out, "out", dtype, dev)
        if y_rows != rows or y_cols != n:
            _shape(out, "out", (rows, n))
        _on_gpu(dev)
        increment_version(out)
        y = out
    mean = torch.empty((rows,), dtype=torch.float32, device=device)
    rstd = torch.empty((rows,), dtype=torch.float32, device=device)
    args = _hip.LayerNorm(_DTYPES[dtype], w_f32, rows, n, eps, x.data_ptr(), ldx, None, 0, w_ptr, b_ptr, y.data_ptr(), ldy, mean.data_ptr(), rstd.data_ptr())
    _call(dev, _hip.load().smrt_layer_norm_forward, C.byref(args))
    return y, mean, rstd


def layer_norm_backward(grad, x, mean, rstd, weight=None, need_x=True, need_weight=True, need_bias=True):
    """Gradients ``(dx, dweight, dbias)`` of ``layer_norm`` from ``grad`` = d loss / d y.  ``x`` is the forward pass's input or its 8-bit form;
    ``mean`` and ``rstd`` are what it returned.  Without a ``weight`` only ``dx`` is computed."""
    dev = _device_of(grad, "grad")
    rows, n, ldg = _matrix(grad, "grad", None, dev)
    dtype, device = grad.dtype, grad.device
    if not 1 <= n <= 32768:
        raise ValueError("layer norm takes 1 to 32768 columns, got %d" % n)
    w_f32, w_ptr, _ = _norm_weight(weight, None, dtype, dev, n)
    x_ptr, ldx, xs_ptr, ld_xs = _kept(x, "x", rows, n, dtype, dev)
    _tensor(mean, "mean", 1, torch.float32, dev)
    _tensor(rstd, "rstd", 1, torch.float32, dev)
    if mean.shape[0] != rows or rstd.shape[0] != rows:
        raise ValueError("mean and rstd must have shape (%d,), got %r and %r" % (rows, tuple(mean.shape), tuple(rstd.shape)))
    _on_gpu(dev)
    dx = grad.new_empty((rows, n)) if need_x else None
    dw = weight.new_empty((n,)) if need_weight and weight is not None else None
    db = weight.new_empty((n,)) if need_bias and weight is not None else None
    args = _hip.LayerNorm(_DTYPES[dtype], w_f32, rows, n, 0.0, x_ptr, ldx, xs_ptr, ld_xs, w_ptr, None, None, 0, mean.data_ptr(), rstd.data_ptr(),
                          grad.data_ptr(), ldg, None if dx is None else dx.data_ptr(), n, None if dw is None else dw.data_ptr(),
                          None if db is None else db.data_ptr())
    lib, ref = _hip.load(), C.byref(args)
    size = lib.smrt_layer_norm_backward_workspace(ref)
    work = torch.empty((size,), dtype=torch.uint8, device=device) if size > 0 else None
    _call(dev, lib.smrt_layer_norm_backward, ref, None if work is None else work.data_ptr(), size)
    return dx, dw, db
