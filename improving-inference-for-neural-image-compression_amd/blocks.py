"""Token blocks: matrix product with a fused epilogue, layer norm and counter-based dropout on the device, forward and backward
(include/sga_hip.h: sga_op_linear_*, sga_op_layer_norm_*, sga_op_dropout).

A token is a row: the last dimension holds the features, all others are tokens -- `[B, yh, yw, C]` latents as they come out of
`SGACodec.encode` are B * yh * yw tokens of C features.  A pre-norm block and its gradient:

    h, mean, rstd = layer_norm(x, nw, nb, want_stats=True)
    a, pre = linear(h, w1, b1, act="gelu", want_pre=True)
    y = linear(a, w2, b2, residual=x, dropout=(0.1, seed, layer))

    g_a, g_w2, g_b2 = linear_grad(g_y, a, w2, dropout=(0.1, seed, layer))
    g_h, g_w1, g_b1 = linear_grad(g_a, h, w1, pre=pre, act="gelu")
    g_x, g_nw, g_nb = layer_norm_grad(g_h, x, mean, rstd, nw, g_add=g_y)

float32, bfloat16 or float16 tensors of one device; sums and statistics in float32, one rounding on store.  The last dimension has
stride 1, the dimensions before it one common stride (a slice of a wider buffer, an expanded row); anything else is
refused, not copied.  Calls run on the current stream of the tensors' device and take their outputs and workspace from torch's
allocator, so they may be captured into a graph; results carry no autograd history, but a tensor written through `out` counts
as changed in place: autograd refuses a backward pass that needs what it held, and an `out` that requires a gradient is refused.  `dropout` is (p, seed, offset), or (p, state) with `state` an int64 tensor
{seed, offset} on the device that is read when the kernel runs (a captured graph draws new numbers when it changes).
There is no CPU path.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _lib

ACTIVATIONS = tuple(_lib.ACTS)
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_U64 = (1 << 64) - 1
_Tensor = torch.Tensor
_empty = torch.empty
_empty_like = torch.empty_like

# The argument structures as bytes: a call is a few microseconds long, and filling a ctypes structure would be half of it.
_DROP = "dQQP"
_LINEAR = struct.Struct("@q4i PqPqPPqPqP Pq PPP " + _DROP).pack
_NORM = struct.Struct("@q3if PqPP PPP PqPq PPP").pack
_DROPOUT = struct.Struct("@" + _DROP).pack
_NO_DROP = (0.0, 0, 0, 0)
_NOMEM = -6
_entry = {}


def _rows(t, what, dtype=None, device=None, features=None):
    """-> (rows, features, row stride) of a tensor whose leading dimensions collapse into one."""
    if isinstance(t, _Tensor) and t.is_cuda and t.is_contiguous() and (device is None or t.device == device):
        shape = t.shape
        if (t.dtype is dtype if dtype is not None else t.dtype in _DTYPES) and len(shape) and shape[-1]:
            n = shape[-1]
            if features is None or n == features:
                return t.numel() // n, n, n
    return _rows_of_any(t, what, dtype, device, features)


def _rows_of_any(t, what, dtype, device, features):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s: a tensor is expected, got %s" % (what, type(t).__name__))
    if t.dtype not in _DTYPES or (dtype is not None and t.dtype != dtype):
        raise TypeError("%s: %s is expected, got %s" % (what, dtype or "float32, bfloat16 or float16", t.dtype))
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError("%s: at least one feature is expected, got shape %s" % (what, tuple(t.shape)))
    n = t.shape[-1]
    if features is not None and n != features:
        raise ValueError("%s has %d features, %d are expected" % (what, n, features))
    if n > 1 and t.stride(-1) != 1:
        raise ValueError("%s: the features have to be adjacent (stride 1), got strides %s" % (what, t.stride()))
    rows, ld = t.numel() // n, None
    if rows > 1:
        dims = [(s, k) for s, k in zip(t.shape[:-1], t.stride()[:-1]) if s != 1]
        for (_, outer), (s, inner) in zip(dims, dims[1:]):
            if outer != s * inner:
                raise ValueError("%s: the rows have no common stride (shape %s, strides %s): call .contiguous() first"
                                 % (what, tuple(t.shape), t.stride()))
        ld = dims[-1][1]
        if ld != 0 and ld < n:
            raise ValueError("%s: rows overlap (row stride %d, %d features)" % (what, ld, n))
    if t.device.type != "cuda":
        raise ValueError("%s: a tensor on the GPU is expected, this one is on %s" % (what, t.device))
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, the other tensors on %s" % (what, t.device, device))
    return rows, n, n if ld is None else ld


def _vector(t, what, n, dtypes, device):
    if t is None:
        return 0
    if isinstance(t, _Tensor) and t.dtype in dtypes and t.shape == (n,) and t.is_contiguous() and t.device == device:
        return t.data_ptr()
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        raise TypeError("%s: a tensor of %s is expected" % (what, " or ".join(str(d) for d in dtypes)))
    if t.device != device or tuple(t.shape) != (n,) or not t.is_contiguous():
        raise ValueError("%s: %d adjacent values on %s are expected, got %s on %s" % (what, n, device, tuple(t.shape), t.device))
    return t.data_ptr()


def _param_type(weight, bias, dt):
    """The type of a norm's parameters: weight's (bias's without a weight), which is x's type `dt` or float32; `dt` where there are none."""
    t, what = (weight, "weight") if weight is not None else (bias, "bias")
    if t is None:
        return dt
    if not isinstance(t, _Tensor):
        raise TypeError("%s: a tensor is expected, got %s" % (what, type(t).__name__))
    if t.dtype != dt and t.dtype != torch.float32:
        raise TypeError("%s: %s or torch.float32 is expected, got %s" % (what, dt, t.dtype))
    return t.dtype


def _like(x):
    """A tensor for a result of x's shape and type (rows without gaps)."""
    return _empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _same(t, like, what):
    if t.shape != like:
        raise ValueError("%s has shape %s, %s is expected" % (what, tuple(t.shape), tuple(like)))


def _apart(out, rows, n, ld, t, what, t_rows, t_n, t_ld):
    """Refuses an output whose memory overlaps an input's; columns side by side in one buffer do not."""
    if t is None or not rows or not t_rows:
        return
    e = out.element_size()
    a, c = out.data_ptr() // e, t.data_ptr() // e
    if a < c + (t_rows - 1) * t_ld + t_n and c < a + (rows - 1) * ld + n:
        side = (a - c) % ld
        if ld != t_ld or side < t_n or side + n > ld:
            raise ValueError("out overlaps %s" % what)


def _contiguous(t, what):
    if not t.is_contiguous():
        raise ValueError("%s has to be contiguous" % what)
    return t.data_ptr()


def _drop(dropout, device):
    """-> the members of sga_dropout"""
    if dropout is None:
        return _NO_DROP
    p = float(dropout[0])
    if not 0.0 <= p <= 1.0:
        raise ValueError("dropout: a probability is expected, got %r" % (dropout[0],))
    if len(dropout) == 2 and isinstance(dropout[1], _Tensor):
        s = dropout[1]
        if s.dtype != torch.int64 or s.numel() != 2 or not s.is_contiguous() or s.device != device:
            raise ValueError("dropout: the state is an int64 tensor {seed, offset} on %s" % device)
        return p, 0, 0, s.data_ptr()
    if len(dropout) != 3:
        raise ValueError("dropout: (p, seed, offset) or (p, state tensor) is expected")
    return p, int(dropout[1]) & _U64, int(dropout[2]) & _U64, 0


def _act(act):
    try:
        return _lib.ACTS[act]
    except KeyError:
        raise ValueError("act: one of %s is expected, got %r" % (", ".join(ACTIVATIONS), act)) from None


def _call(name, device, *args):
    """An entry point on the device's current stream -> status."""
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(_lib.load_library(), name)
    i = device.index
    if torch._C._cuda_getDevice() == i:
        return fn(*args, torch._C._cuda_getCurrentRawStream(i))
    with torch.cuda.device(i):
        return fn(*args, torch._C._cuda_getCurrentRawStream(i))


def _call_with_workspace(name, a, device, backward):
    """An entry point with the workspace that it asks for; a forward call is first made without one, which most need not have."""
    st = _NOMEM if backward else _call(name, device, a, None, 0)
    if st == _NOMEM:
        need = C.c_int64(0)
        st = getattr(_lib.load_library(), name[:-4] + "_workspace")(a, backward, C.addressof(need))
        if st == 0:
            n = need.value
            ws = _empty(n, dtype=torch.uint8, device=device) if n else None
            st = _call(name, device, a, ws.data_ptr() if n else None, n)
    if st:
        _lib.check(None, None, st, name)


def linear(x, weight, bias=None, act="none", residual=None, dropout=None, want_pre=False, out=None):
    """residual + D_p(act(x weight^T + bias)): x [..., K], weight [N, K], bias [N], residual [..., N] -> [..., N].

    want_pre: -> (out, pre), pre = x weight^T + bias, which `linear_grad` needs where there is an activation.  out: a tensor to write
    to (it may be `residual` itself, to add in place)."""
    rows, k, ld_x = _rows(x, "x")
    dt, dev = x.dtype, x.device
    n, _, ld_w = _rows(weight, "weight", dt, dev, k)
    if weight.dim() != 2:
        raise ValueError("weight: [out_features, in_features] is expected, got shape %s" % (tuple(weight.shape),))
    shape = x.shape[:-1] + (n,)
    p_bias = _vector(bias, "bias", n, (dt,), dev)
    ld_res, ld_out, p_res, p_pre, pre = n, n, 0, 0, None
    if residual is not None:
        _, _, ld_res = _rows(residual, "residual", dt, dev, n)
        _same(residual, shape, "residual")
        p_res = residual.data_ptr()
    given = out is not None
    if not given:
        out = x.new_empty(shape)
    else:
        _, _, ld_out = _rows(out, "out", dt, dev, n)
        _same(out, shape, "out")
        if ld_out == 0 and rows > 1:
            raise ValueError("out: its rows overlap")
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("out requires a gradient, which the call would not record")
        _apart(out, rows, n, ld_out, x, "x", rows, k, ld_x)
        _apart(out, rows, n, ld_out, weight, "weight", n, k, ld_w)
        _apart(out, rows, n, ld_out, bias, "bias", 1, n, n)
        if p_res != out.data_ptr() or ld_res != ld_out:
            _apart(out, rows, n, ld_out, residual, "residual", rows, n, ld_res)
    if want_pre:
        pre = x.new_empty(shape)
        p_pre = pre.data_ptr()
    a = _LINEAR(rows, k, n, _DTYPES[dt], _act(act), x.data_ptr(), ld_x, weight.data_ptr(), ld_w, p_bias, p_res, ld_res,
                out.data_ptr(), ld_out, p_pre, 0, 0, 0, 0, 0, *_drop(dropout, dev))
    _call_with_workspace("sga_op_linear_fwd", a, dev, 0)
    if given:
        torch.autograd.graph.increment_version(out)
    return (out, pre) if want_pre else out


def linear_grad(g_out, x, weight, pre=None, act="none", dropout=None, want=(True, True, True)):
    """The gradients of `linear` -> (g_x, g_weight, g_bias), None where `want` is false.  The gradient of the residual is g_out."""
    rows, n, ld_g = _rows(g_out, "g_out")
    dt, dev = g_out.dtype, g_out.device
    rx, k, ld_x = _rows(x, "x", dt, dev)
    nw, _, ld_w = _rows(weight, "weight", dt, dev, k)
    if weight.dim() != 2 or nw != n:
        raise ValueError("weight: [%d, %d] is expected, got shape %s" % (n, k, tuple(weight.shape)))
    _same(g_out, x.shape[:-1] + (n,), "g_out")
    code = _act(act)
    if code:
        if pre is None:
            raise ValueError("pre: the value before the activation is needed for act=%r" % act)
        _rows(pre, "pre", dt, dev, n)
        _same(pre, g_out.shape, "pre")
        _contiguous(pre, "pre")
    g_x = _like(x) if want[0] else None
    g_w = _empty((n, k), dtype=dt, device=dev) if want[1] else None
    g_b = _empty(n, dtype=dt, device=dev) if want[2] else None
    a = _LINEAR(rows, k, n, _DTYPES[dt], code, x.data_ptr(), ld_x, weight.data_ptr(), ld_w, 0, 0, 0, 0, 0, pre.data_ptr() if code else 0,
                g_out.data_ptr(), ld_g, g_x.data_ptr() if want[0] else 0, g_w.data_ptr() if want[1] else 0, g_b.data_ptr() if want[2] else 0,
                *_drop(dropout, dev))
    _call_with_workspace("sga_op_linear_bwd", a, dev, 1)
    return g_x, g_w, g_b


def layer_norm(x, weight=None, bias=None, eps=1e-5, want_stats=False):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension; weight and bias [C] in x's type or float32.

    want_stats: -> (y, mean, rstd), the last two float32 of x's leading shape, which `layer_norm_grad` needs."""
    rows, n, ld = _rows(x, "x")
    dt, dev = x.dtype, x.device
    pt = _param_type(weight, bias, dt)
    w, b = _vector(weight, "weight", n, (pt,), dev), _vector(bias, "bias", n, (pt,), dev)
    if not eps >= 0.0:
        raise ValueError("eps: a number >= 0 is expected, got %r" % (eps,))
    y = _like(x)
    mean = rstd = None
    p_mean = p_rstd = 0
    if want_stats:
        mean = _empty(x.shape[:-1], dtype=torch.float32, device=dev)
        rstd = _empty_like(mean)
        p_mean, p_rstd = mean.data_ptr(), rstd.data_ptr()
    st = _call("sga_op_layer_norm_fwd", dev, _NORM(rows, n, _DTYPES[dt], _DTYPES[pt], eps, x.data_ptr(), ld, w, b, y.data_ptr(), p_mean, p_rstd,
                                                   0, 0, 0, 0, 0, 0, 0))
    if st:
        _lib.check(None, None, st, "sga_op_layer_norm_fwd")
    return (y, mean, rstd) if want_stats else y


def layer_norm_grad(g_y, x, mean, rstd, weight=None, g_add=None, want=(True, True, True), param_dtype=None):
    """The gradients of `layer_norm` -> (g_x, g_weight, g_bias), None where `want` is false; g_x has `g_add`, the gradient that reaches
    x past the norm, added.  g_weight and g_bias have weight's type (without a weight: param_dtype, x's type unless given)."""
    rows, n, ld = _rows(x, "x")
    dt, dev = x.dtype, x.device
    _, _, ld_g = _rows(g_y, "g_y", dt, dev, n)
    _same(g_y, x.shape, "g_y")
    for t, what in ((mean, "mean"), (rstd, "rstd")):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != dev or t.numel() != rows:
            raise ValueError("%s: %d float32 values on %s are expected" % (what, rows, dev))
        _contiguous(t, what)
    ld_add = n
    if g_add is not None:
        _, _, ld_add = _rows(g_add, "g_add", dt, dev, n)
        _same(g_add, x.shape, "g_add")
    w = _vector(weight, "weight", n, (dt, torch.float32), dev)
    pt = weight.dtype if weight is not None else param_dtype or dt
    if pt not in (dt, torch.float32):
        raise TypeError("param_dtype: %s or torch.float32 is expected, got %s" % (dt, pt))
    g_x = _like(x) if want[0] else None
    g_w = _empty(n, dtype=pt, device=dev) if want[1] else None
    g_b = _empty(n, dtype=pt, device=dev) if want[2] else None
    a = _NORM(rows, n, _DTYPES[dt], _DTYPES[pt], 0.0, x.data_ptr(), ld, w, 0, 0, mean.data_ptr(), rstd.data_ptr(), g_y.data_ptr(), ld_g,
              g_add.data_ptr() if g_add is not None else 0, ld_add, g_x.data_ptr() if want[0] else 0, g_w.data_ptr() if want[1] else 0,
              g_b.data_ptr() if want[2] else 0)
    _call_with_workspace("sga_op_layer_norm_bwd", a, dev, 1)
    return g_x, g_w, g_b


def dropout(x, p, seed, offset=0, residual=None):
    """residual + D_p(x).  seed: an int, or the int64 state tensor {seed, offset} on the device.  The gradient w.r.t. x is the same
    call on the gradient (without residual); the mask is that of a `linear` with the same p, seed, offset and output shape."""
    rows, n, ld = _rows(x, "x")
    dt, dev = x.dtype, x.device
    ld_res = n
    if residual is not None:
        _, _, ld_res = _rows(residual, "residual", dt, dev, n)
        _same(residual, x.shape, "residual")
    d = _DROPOUT(*_drop((p, seed) if isinstance(seed, _Tensor) else (p, seed, offset), dev))
    y = _like(x)
    st = _call("sga_op_dropout", dev, x.data_ptr(), ld, residual.data_ptr() if residual is not None else None, ld_res, y.data_ptr(), rows, n,
               _DTYPES[dt], d)
    if st:
        _lib.check(None, None, st, "sga_op_dropout")
    return y
