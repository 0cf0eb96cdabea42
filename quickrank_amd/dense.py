"""Dense operators of a neural document scorer on torch tensors: layer norm, dropout and the gated
feed-forward unit, with their gradients (include/qr_hip.h, "dense operators").

Every call runs the HIP kernels of libqr_hip.so on the tensors' own device, on torch's current
stream of that device, and only enqueues; tensors used on another stream than the one they were
made on need `Tensor.record_stream`, as with any torch operator.  Gradients are explicit calls, as
the lambda pass is one: nothing is recorded by autograd, so a tensor that requires a gradient is
refused while autograd records, and one with a forward-mode tangent always.

A tensor of rows is f32, bf16 or f16 and is read as a matrix of its last dimension: 2-D with any
row stride (0 included), or contiguous with any leading dimensions.
"""
import ctypes as C
from operator import index

import torch
from torch.autograd import forward_ad

from ._capi import QrError, lib

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3, "sigmoid": 4}


def _fail(rc):
    raise QrError(f"{lib().qr_last_error(None).decode()} (code {rc})", rc)


def _refuse(msg):
    raise QrError(msg, 3)


_stream = torch._C._cuda_getCurrentRawStream


def _check(t, what, device=None):
    """The tensor's device number, of `device` where that is given."""
    if not isinstance(t, torch.Tensor) or t.dtype not in TYPES:
        _refuse(f"{what} is a torch tensor of f32, bf16 or f16")
    if t.requires_grad and torch.is_grad_enabled():
        _refuse(f"{what} requires a gradient, which this call would not record: use torch.no_grad() and the "
                "backward call")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        _refuse(f"{what} has a forward-mode tangent, which this call would lose")
    if t.is_neg():
        _refuse(f"{what} is a view whose numbers are negated when read: use resolve_neg()")
    at = t.get_device()
    if at < 0 or not t.is_cuda:
        _refuse(f"{what} is not on a GPU: there is no CPU fallback")
    if device is not None and at != device:
        _refuse(f"{what} is on {t.device}, not on cuda:{device}")
    return at


def _empty(x):
    """A contiguous tensor of the shape and type of x."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _rows(t, what, device=None):
    """(rows, cols, stride, device) of a tensor read as a matrix of its last dimension."""
    at = _check(t, what, device)
    shape = t.shape
    if not shape:
        _refuse(f"{what} has no dimension")
    cols = shape[-1]
    if t.is_contiguous():
        return (t.numel() // cols if cols else 0), cols, cols, at
    if len(shape) == 2 and (t.stride(1) == 1 or cols == 1):
        return shape[0], cols, t.stride(0) if shape[0] > 1 else cols, at
    _refuse(f"{what} is neither contiguous nor a matrix of contiguous rows")


def _same(t, what, like, of, device):
    """The stride of a tensor that has to match another's shape and type."""
    if isinstance(t, torch.Tensor) and (t.shape != like.shape or t.dtype != like.dtype):
        _refuse(f"{what} has another shape or type than {of}")
    return _rows(t, what, device)[2]


def _vector(t, what, x, cols, device):
    if t is None:
        return None
    _check(t, what, device)
    if t.shape != (cols,) or not t.is_contiguous():
        _refuse(f"{what} is a contiguous vector of the rows' length")
    if t.dtype != torch.float32 and t.dtype != x.dtype:
        _refuse(f"{what} has the rows' type or f32")
    return t.data_ptr()


def _stat(t, what, rows, device):
    _check(t, what, device)
    if t.dtype != torch.float32 or t.numel() != rows or not t.is_contiguous():
        _refuse(f"{what} is contiguous f32, one value a row")
    return t.data_ptr()


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(y, mean, rstd): y = (x - mean) * rstd * weight + bias over the last dimension; mean and rstd f32
    [rows], what layer_norm_backward takes.  weight / bias: the rows' type or f32, both alike."""
    rows, cols, ld, at = _rows(x, "x")
    if cols == 0:
        _refuse("layer norm: rows of no columns")
    w, b = _vector(weight, "weight", x, cols, at), _vector(bias, "bias", x, cols, at)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        _refuse("weight and bias have two types")
    p = weight if weight is not None else bias if bias is not None else x
    y, mean = _empty(x), x.new_empty(rows, dtype=torch.float32)
    rstd = torch.empty_like(mean)
    rc = lib().qr_layer_norm_async(at, _stream(at), TYPES[x.dtype], TYPES[p.dtype], rows, cols, x.data_ptr(), ld, w, b, eps,
                                   y.data_ptr(), cols, mean.data_ptr(), rstd.data_ptr())
    if rc:
        _fail(rc)
    return y, mean, rstd


def layer_norm_backward(dy, x, weight, mean, rstd, param_dtype=None):
    """(dx, dweight, dbias) of layer_norm; the last two in the weight's type (weight None: param_dtype,
    by default the rows')."""
    rows, cols, ldx, at = _rows(x, "x")
    lddy = _same(dy, "dy", x, "x", at)
    if cols == 0:
        _refuse("layer norm backward: rows of no columns")
    w = _vector(weight, "weight", x, cols, at)
    pt = weight.dtype if weight is not None else param_dtype or x.dtype
    if pt != x.dtype and pt != torch.float32:
        _refuse("weight and bias have the rows' type or f32")
    m, r = _stat(mean, "mean", rows, at), _stat(rstd, "rstd", rows, at)
    dx, dweight = _empty(x), torch.empty_like(weight) if weight is not None else x.new_empty(cols, dtype=pt)
    dbias = torch.empty_like(dweight)
    need = C.c_size_t()
    rc = lib().qr_layer_norm_backward_workspace(rows, cols, C.byref(need))
    ws = x.new_empty(need.value, dtype=torch.uint8)
    rc = rc or lib().qr_layer_norm_backward_async(
        at, _stream(at), TYPES[x.dtype], TYPES[pt], rows, cols, dy.data_ptr(), lddy, x.data_ptr(), ldx, w, m, r,
        dx.data_ptr(), cols, dweight.data_ptr(), dbias.data_ptr(), ws.data_ptr(), need.value)
    if rc:
        _fail(rc)
    return dx, dweight, dbias


def _dropout(x, p, seed, offset, residual, counter):
    rows, cols, ld, at = _rows(x, "x")
    ldr = _same(residual, "residual", x, "x", at) if residual is not None else 0
    if counter is not None and not (isinstance(counter, torch.Tensor) and counter.dtype == torch.int64
                                    and counter.numel() == 1 and counter.device == x.device):
        _refuse("counter is one int64 on the device of x")
    if not 0.0 <= p <= 1.0:
        _refuse("dropout: p is a number of 0 to 1")
    try:
        seed, offset = index(seed) & 0xFFFFFFFFFFFFFFFF, index(offset) & 0xFFFFFFFFFFFFFFFF
    except TypeError:
        _refuse("dropout: seed and offset are whole numbers")
    y = _empty(x)
    rc = lib().qr_dropout_async(at, _stream(at), TYPES[x.dtype], rows, cols, x.data_ptr(), ld,
                                residual.data_ptr() if residual is not None else None, ldr, y.data_ptr(), cols, p,
                                seed, offset,
                                counter.data_ptr() if counter is not None else None)
    if rc:
        _fail(rc)
    return y


def dropout(x, p, seed, offset=0, residual=None, counter=None):
    """residual + (kept ? x / (1 - p) : 0), the mask a function of (seed, offset, element) that is never
    stored.  A call uses dropout_words(x) numbers of its seed from `offset` on; counter: an int64 on the
    device that is added to `offset` when the kernel runs (a captured graph draws anew at each replay)."""
    return _dropout(x, p, seed, offset, residual, counter)


def dropout_backward(dy, p, seed, offset=0, counter=None):
    """The gradient of dropout's x (that of its residual is dy)."""
    return _dropout(dy, p, seed, offset, None, counter)


def dropout_words(x):
    """How far `offset` moves from one call to the next of the same seed."""
    return (x.numel() + 3) // 4


def _weights(x, k, w_gate, w_up, device):
    _check(w_gate, "w_gate", device)
    _check(w_up, "w_up", device)
    shape, stride, other = w_gate.shape, w_gate.stride(), w_up.stride()
    if len(shape) != 2 or shape[1] != k or w_gate.dtype != x.dtype or (stride[1] != 1 and k > 1):
        _refuse("w_gate is a matrix of contiguous rows, [n][columns of x], of the type of x")
    # (the kernels read both by one row stride; the stride of a dimension of one element is not read)
    if w_up.shape != shape or w_up.dtype != x.dtype or (other[1] != 1 and k > 1) or (other[0] != stride[0] and shape[0] > 1):
        _refuse("w_up differs from w_gate in shape, stride or type")
    if k == 0 or shape[0] == 0:
        _refuse("gated ffn: no columns")
    return shape[0], stride[0] if shape[0] > 1 else k


def _act(act):
    if act not in ACTS:
        _refuse(f"unknown activation {act!r}: one of {', '.join(ACTS)}")
    return ACTS[act]


def gated_ffn(x, w_gate, w_up, act="silu", save=False):
    """act(x @ w_gate.T) * (x @ w_up.T); save=True: (that, gate, up), the two products that
    gated_ffn_backward takes."""
    m, k, ldx, at = _rows(x, "x")
    n, ldw = _weights(x, k, w_gate, w_up, at)
    a = _act(act)
    shape = x.shape[:-1] + (n,)
    h = x.new_empty(shape)
    g, u = (torch.empty_like(h), torch.empty_like(h)) if save else (None, None)
    px, pg, pu, e = x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), x.element_size()
    ws, need, rc = None, C.c_size_t(), 0
    # rows that do not start and end at 16-byte boundaries or lie more than 4 MB apart are copied first
    if (px | pg | pu | ldx * e | ldw * e | k * e) & 15 or max(ldx, ldw) * e > 1 << 22:
        rc = lib().qr_gated_ffn_workspace(TYPES[x.dtype], m, k, n, C.byref(need))
        ws = x.new_empty(need.value, dtype=torch.uint8)
    rc = rc or lib().qr_gated_ffn_async(at, _stream(at), TYPES[x.dtype], a, m, k, n, px, ldx, pg, pu, ldw, h.data_ptr(), n,
                                        g.data_ptr() if save else None, u.data_ptr() if save else None,
                                        ws.data_ptr() if ws is not None else None, need.value)
    if rc:
        _fail(rc)
    return (h, g, u) if save else h


def gated_ffn_backward(dh, x, w_gate, w_up, gate, up, act="silu"):
    """(dx, dw_gate, dw_up) of gated_ffn from its saved products."""
    m, k, ldx, at = _rows(x, "x")
    n, ldw = _weights(x, k, w_gate, w_up, at)
    a = _act(act)
    for t, what in ((dh, "dh"), (gate, "gate"), (up, "up")):
        if not isinstance(t, torch.Tensor) or t.shape != x.shape[:-1] + (n,) or t.dtype != x.dtype:
            _refuse(f"{what} has another shape or type than the forward call's result")
        _check(t, what, at)
    if not gate.is_contiguous() or not up.is_contiguous():
        _refuse("gate and up are contiguous, as the forward call returns them")
    lddh = _rows(dh, "dh")[2]
    dx, dw_gate = _empty(x), x.new_empty((n, k))
    dw_up = torch.empty_like(dw_gate)
    need = C.c_size_t()
    rc = lib().qr_gated_ffn_backward_workspace(TYPES[x.dtype], m, k, n, C.byref(need))
    ws = x.new_empty(need.value, dtype=torch.uint8)
    rc = rc or lib().qr_gated_ffn_backward_async(
        at, _stream(at), TYPES[x.dtype], a, m, k, n, dh.data_ptr(), lddh, x.data_ptr(), ldx, w_gate.data_ptr(),
        w_up.data_ptr(), ldw, gate.data_ptr(), up.data_ptr(), dx.data_ptr(), k, dw_gate.data_ptr(), dw_up.data_ptr(),
        ws.data_ptr(), need.value)
    if rc:
        _fail(rc)
    return dx, dw_gate, dw_up
