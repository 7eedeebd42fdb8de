"""Matrix products with bias, activation and residual in one launch: the 1x1 convolutions of the detection head
(object_detection/yolov5/models/yolo.py:41,52) and of the blocks before it, on channel-major maps, and the same operator on rows.

  y = act(W x + b) + residual

Sums, bias, activation and residual are fp32 and the result is rounded once.  All three entries are differentiable (x, weight,
bias, residual) and take fp32, fp16 or bf16 tensors of one type; under torch.autocast their inputs are cast to its type, as
torch's own layers do.  The backward of an activation reads the pre-activation, kept in the tensors' type.  A second derivative is
not offered.
"""
import ctypes
import struct

import torch

from . import _lib as L

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "sigmoid": 4}
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_PRODUCTS = 5


class Product(ctypes.Structure):
    """Mirror of dh_product in include/dethead.h."""
    _fields_ = ([(n, L.c_void_p) for n in ("a", "b", "bias", "residual", "out", "z", "a_sum")]
                + [(n, L.c_i64) for n in ("lda", "ldb", "ldo", "ldr", "a_batch", "b_batch", "o_batch", "res_batch")]
                + [(n, L.c_int) for n in ("I", "J", "R", "batch", "a_by_reduction", "b_by_reduction", "bias_on_i", "reduce_batch")])


# The same struct as bytes, its fields in order: a call fills it an order of magnitude faster than ctypes' attributes.
_pack = struct.Struct("7Q8q8i").pack
assert struct.calcsize("7Q8q8i") == ctypes.sizeof(Product)


def _run(products, dtype, activation, device):
    """One launch of the given packed products."""
    n, table, code, lib = len(products), b"".join(products), _DTYPES[dtype], L.lib()
    need = lib.dh_products_workspace(table, n, code)
    ws = L.workspace(need, device) if need else None
    with L.device_guard(device):
        L.check(lib.dh_products(table, n, code, activation, ws.data_ptr() if need else None, need, L.raw_stream()), "dh_products")


def _slope(dy, z, activation, want_bias, outer, n, inner):
    """(dz, dbias): dy times the activation's derivative (dy itself without one) and its sum for the bias."""
    dz = torch.empty_like(dy) if z is not None else dy
    if z is None and not want_bias:
        return dz, None
    dbias = torch.empty(n, dtype=dy.dtype, device=dy.device) if want_bias else None
    lib = L.lib()
    need = lib.dh_product_slope_workspace(n) if want_bias else 0
    ws = L.workspace(need, dy.device) if want_bias else None
    with L.device_guard(dy.device):
        L.check(lib.dh_product_slope(dy.data_ptr(), z.data_ptr() if z is not None else None, dz.data_ptr(),
                                     dbias.data_ptr() if want_bias else None, outer, n, inner, activation, _DTYPES[dy.dtype],
                                     ws.data_ptr() if want_bias else None, need, L.raw_stream()), "dh_product_slope")
    return dz, dbias


# ---- layouts: rows (M, K) -> (M, N) and maps (B, K, ny, nx) -> (B, N, ny, nx), both with a dense weight of N x K ----

def _as_rows(t):
    """(..., C) -> (M, C) with the last axis dense and one stride between rows; a copy only where the strides do not allow a
    view (or rows overlap, as in an expanded tensor)."""
    t = t.reshape(t.shape[:-1].numel(), t.shape[-1]) if t.dim() != 2 else t
    if not t.is_contiguous() and (t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _as_planes(t):
    """(B, C, ny, nx) with dense planes, and the distance between its images: a slice of a wider tensor's channels is taken as
    it is, anything else that is not dense is copied."""
    if t.is_contiguous():
        return t, t.shape[1] * t.shape[2] * t.shape[3]
    b, c, h, w = t.shape
    s = t.stride()
    if s[1:] == (h * w, w, 1) and s[0] >= c * h * w:
        return t, s[0]
    return t.contiguous(), c * h * w


def _rows_forward(x, w, bias, res, out, z):
    m, k = x.shape
    n = w.shape[0]
    return _pack(x.data_ptr(), w.data_ptr(), bias.data_ptr() if bias is not None else 0, res.data_ptr() if res is not None else 0,
                 out.data_ptr(), z.data_ptr() if z is not None else 0, 0, x.stride(0) if m > 1 else k, k, n,
                 res.stride(0) if res is not None and m > 1 else n, 0, 0, 0, 0, m, n, k, 1, 1, 1, 0, 0)


def _maps_forward(x, x_batch, w, bias, res, res_batch, out, z):
    b, k, h, v = x.shape
    n, p = w.shape[0], h * v
    return _pack(w.data_ptr(), x.data_ptr(), bias.data_ptr() if bias is not None else 0, res.data_ptr() if res is not None else 0,
                 out.data_ptr(), z.data_ptr() if z is not None else 0, 0, k, p, p, p, 0, x_batch, n * p, res_batch, n, p, k, b, 1, 0, 1, 0)


def _grad_input(rows, dz, w, out):
    n, k = w.shape[0], w.shape[1]
    if rows:
        return _pack(dz.data_ptr(), w.data_ptr(), 0, 0, out.data_ptr(), 0, 0, n, k, k, 0, 0, 0, 0, 0, dz.shape[0], k, n, 1, 1, 0, 0, 0)
    b, p = dz.shape[0], dz.shape[2] * dz.shape[3]
    return _pack(w.data_ptr(), dz.data_ptr(), 0, 0, out.data_ptr(), 0, 0, k, p, p, 0, 0, n * p, k * p, 0, k, p, n, b, 0, 0, 0, 0)


def _grad_weight(rows, dz, x, x_batch, out, dbias):
    """With dbias: the bias gradient beside the weight's, from the same read of dz."""
    k, n, db = x.shape[1], dz.shape[1], dbias.data_ptr() if dbias is not None else 0
    if rows:
        m = x.shape[0]
        return _pack(dz.data_ptr(), x.data_ptr(), 0, 0, out.data_ptr(), 0, db, n, x.stride(0) if m > 1 else k, k, 0, 0, 0, 0, 0, n, k, m, 1,
                     0, 0, 0, 0)
    b, p = x.shape[0], x.shape[2] * x.shape[3]
    return _pack(dz.data_ptr(), x.data_ptr(), 0, 0, out.data_ptr(), 0, db, p, p, k, 0, n * p, x_batch, 0, 0, n, k, p, b, 1, 1, 0, 1)


def _forward(rows, act, items, keep):
    """items: (x, weight, bias, residual), x (M, K) with `rows`, else (B, K, ny, nx) -> outputs; with keep also what a backward
    needs, (x as it was read, pre-activation) of each."""
    outs, kept, products, alive = [], [], [], []
    for x, w, bias, res in items:
        dtype, device, n = x.dtype, x.device, w.shape[0]
        if not w.is_contiguous():
            w = w.contiguous()
        if bias is not None and not bias.is_contiguous():
            bias = bias.contiguous()
        if rows:
            x = _as_rows(x)
            res = _as_rows(res) if res is not None else None
            out = torch.empty((x.shape[0], n), dtype=dtype, device=device)
        else:
            x, x_batch = _as_planes(x)
            res, res_batch = _as_planes(res) if res is not None else (None, 0)
            out = torch.empty((x.shape[0], n, x.shape[2], x.shape[3]), dtype=dtype, device=device)
        z = torch.empty_like(out) if keep and act else None
        products.append(_rows_forward(x, w, bias, res, out, z) if rows else _maps_forward(x, x_batch, w, bias, res, res_batch, out, z))
        outs.append(out)
        kept += (x, w, z) if keep else ()
        alive.append((x, w, bias, res))         # copies live until the launch is queued
    _run(products, dtype, act, device)
    return outs, kept


class _Products(torch.autograd.Function):
    """The products of one launch with their gradients.  tensors: x, weight, bias, residual of each (bias, residual may be None)."""

    @staticmethod
    def forward(ctx, rows, act, *tensors):
        items = [tensors[k:k + 4] for k in range(0, len(tensors), 4)]
        outs, kept = _forward(rows, act, items, True)
        ctx.rows, ctx.act = rows, act
        ctx.save_for_backward(*kept)
        return tuple(outs)

    @staticmethod
    def backward(ctx, *grads):
        # grad mode is on only under create_graph: then the results are marked as having no further derivative
        return (_Products._marked if torch.is_grad_enabled() else _Products._gradients)(ctx, *grads)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def _marked(ctx, *grads):
        return _Products._gradients(ctx, *grads)

    @staticmethod
    def _gradients(ctx, *grads):
        rows, saved, wants = ctx.rows, ctx.saved_tensors, ctx.needs_input_grad
        result, inputs, weights, alive = [None, None], [], [], []
        for k, dy in enumerate(grads):
            x, w, z = saved[3 * k:3 * k + 3]
            want_x, want_w, want_b, want_r = wants[2 + 4 * k:6 + 4 * k]
            dx = dw = db = None
            if dy is None:
                result += [None] * 4
                continue
            dy = dy.contiguous()
            if want_x or want_w or want_b:
                n, at_weight = dy.shape[1], z is None and want_w and x.shape[1] > 0
                outer, inner = dy.shape[0], 1 if rows else dy.shape[2] * dy.shape[3]
                # without an activation dy is dz: the weight's gradient reads it anyway and sums it for the bias
                dz, db = (dy, torch.empty(n, dtype=dy.dtype, device=dy.device) if want_b else None) if at_weight else \
                    _slope(dy, z, ctx.act, want_b, outer, n, inner)
                if want_x:
                    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
                    inputs.append(_grad_input(rows, dz, w, dx))
                if want_w:
                    dw = torch.empty_like(w)
                    weights.append(_grad_weight(rows, dz, x, 0 if rows else _as_planes(x)[1], dw, db if at_weight else None))
                alive.append(dz)
            result += [dx, dw, db, dy if want_r else None]
        for group in (inputs, weights):
            if group:
                _run(group, saved[0].dtype, 0, saved[0].device)
        return tuple(result)


def _apply(rows, act, items):
    if torch.is_grad_enabled():
        tensors = [t for item in items for t in item]
        if any([t is not None and t.requires_grad for t in tensors]):
            return _Products.apply(rows, act, *tensors)
    return _forward(rows, act, items, False)[0]


def _activation(name, where):
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"{where}: activation must be one of {list(ACTIVATIONS)}, got {name!r}") from None


def _checked(where, x, weight, bias, residual):
    """The four tensors, of one supported type on one ROCm device (cast to autocast's type where that is on)."""
    tensors = [t for t in (x, weight, bias, residual) if t is not None]
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{where}: expected torch.Tensor, got {type(t).__name__}")
    if x is None or weight is None:
        raise TypeError(f"{where}: x and weight must be tensors")
    device = x.get_device()
    if device < 0 or not x.is_cuda:
        raise RuntimeError(f"{where}: x is on {x.device}: object_detection_amd only runs on ROCm devices (no CPU fallback)")
    for t in tensors:
        if t.get_device() != device:
            raise RuntimeError(f"{where}: tensors on {t.device} and {x.device}")
    if torch.is_autocast_enabled("cuda"):
        to = torch.get_autocast_dtype("cuda")
        x, weight, bias, residual = [t.to(to) if t is not None and t.is_floating_point() else t for t in (x, weight, bias, residual)]
        tensors = [t for t in (x, weight, bias, residual) if t is not None]
    dtype = x.dtype
    for t in tensors:
        if t.dtype != dtype or dtype not in _DTYPES:
            raise RuntimeError(f"{where}: x, weight, bias and residual must have one type, fp32, fp16 or bf16; got {t.dtype} and {dtype}")
    return x, weight, bias, residual


def _check_weight(where, weight, bias, inputs):
    shape = weight.shape
    if len(shape) not in (2, 4) or shape[1] != inputs or (len(shape) == 4 and shape[2:] != (1, 1)):
        raise RuntimeError(f"{where}: weight must be (outputs, {inputs}) or (outputs, {inputs}, 1, 1), got {tuple(shape)}")
    if bias is not None and bias.shape != shape[:1]:
        raise RuntimeError(f"{where}: bias must be ({shape[0]},), got {tuple(bias.shape)}")


def linear(x, weight, bias=None, activation=None, residual=None):
    """act(x weight^T + bias) + residual for x (..., C), weight (N, C), bias (N,), residual (..., N) -> (..., N).

    activation: None, "relu", "silu", "gelu" (the exact one, with erf) or "sigmoid".  From one row to many; rows of x and of the
    residual may be strided (a slice of a wider tensor is read in place)."""
    act = _activation(activation, "linear")
    x, weight, bias, residual = _checked("linear", x, weight, bias, residual)
    if x.dim() < 1 or weight.dim() != 2:
        raise RuntimeError(f"linear: x must be (..., C) and weight (N, C), got {tuple(x.shape)} and {tuple(weight.shape)}")
    _check_weight("linear", weight, bias, x.shape[-1])
    if residual is not None and residual.shape != x.shape[:-1] + weight.shape[:1]:
        raise RuntimeError(f"linear: residual must be {tuple(x.shape[:-1] + weight.shape[:1])}, got {tuple(residual.shape)}")
    if x.dim() == 2:
        return _apply(True, act, [(x, weight, bias, residual)])[0]
    rows, n = x.shape[:-1].numel(), weight.shape[0]
    out = _apply(True, act, [(x.reshape(rows, x.shape[-1]), weight, bias, residual.reshape(rows, n) if residual is not None else None)])[0]
    return out.view(x.shape[:-1] + (n,))


def pointwise_conv(x, weight, bias=None, activation=None, residual=None):
    """A 1x1 convolution with its epilogue: act(conv(x) + bias) + residual for x (B, C, ny, nx), weight (N, C) or (N, C, 1, 1),
    bias (N,), residual (B, N, ny, nx) -> (B, N, ny, nx).

    activation as in linear().  A channels_last x runs as rows and gives a channels_last result."""
    act = _activation(activation, "pointwise_conv")
    x, weight, bias, residual = _checked("pointwise_conv", x, weight, bias, residual)
    if x.dim() != 4:
        raise RuntimeError(f"pointwise_conv: x must be (B, C, ny, nx), got {tuple(x.shape)}")
    _check_weight("pointwise_conv", weight, bias, x.shape[1])
    b, c, h, w = x.shape
    n = weight.shape[0]
    if residual is not None and residual.shape != (b, n, h, w):
        raise RuntimeError(f"pointwise_conv: residual must be {(b, n, h, w)}, got {tuple(residual.shape)}")
    if not x.is_contiguous() and x.is_contiguous(memory_format=torch.channels_last):
        res = residual.permute(0, 2, 3, 1).reshape(b * h * w, n) if residual is not None else None
        out = _apply(True, act, [(x.permute(0, 2, 3, 1).reshape(b * h * w, c), weight, bias, res)])[0]
        return out.view(b, h, w, n).permute(0, 3, 1, 2)
    return _apply(False, act, [(x, weight, bias, residual)])[0]


def head_convs(xs, weights, biases):
    """The 1x1 convolutions of a detection head, all levels in one launch (yolo.py:52): xs[l] (B, C_l, ny_l, nx_l), weights[l]
    (N, C_l, 1, 1) or (N, C_l), biases[l] (N,) or None -> the list of (B, N, ny_l, nx_l).  At most five levels."""
    xs, weights, biases = list(xs), list(weights), list(biases)
    if not xs or len(xs) > MAX_PRODUCTS or len(weights) != len(xs) or len(biases) != len(xs):
        raise RuntimeError(f"head_convs: 1 to {MAX_PRODUCTS} levels with a weight and a bias each, got {len(xs)}, {len(weights)}, {len(biases)}")
    items = []
    for x, weight, bias in zip(xs, weights, biases):
        x, weight, bias, _ = _checked("head_convs", x, weight, bias, None)
        if x.dim() != 4:
            raise RuntimeError(f"head_convs, level {len(items)}: x must be (B, C, ny, nx), got {tuple(x.shape)}")
        _check_weight("head_convs", weight, bias, x.shape[1])
        if items and (x.dtype != items[0][0].dtype or x.get_device() != items[0][0].get_device()):
            raise RuntimeError(f"head_convs, level {len(items)}: {x.dtype} on {x.device}, level 0 {items[0][0].dtype} on {items[0][0].device}")
        items.append((x, weight, bias, None))
    return list(_apply(False, 0, items))
