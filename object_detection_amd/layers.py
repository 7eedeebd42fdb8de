"""Matrix products with bias, activation and residual in one launch: the 1x1 convolutions of the detection head
(object_detection/yolov5/models/yolo.py:41,52) and of the blocks before it, on channel-major maps, and the same operator on rows.

  y = act(W x + b) + residual

Sums, bias, activation and residual are fp32 and the result is rounded once.  All three entries are differentiable (x, weight,
bias, residual) and take fp32, fp16 or bf16 tensors of one type; under torch.autocast their inputs are cast to its type, as
torch's own layers do.  A second derivative is not offered.
"""
import ctypes

import torch

from . import _lib as L

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "sigmoid": 4}
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_PRODUCTS = 5


class Product(ctypes.Structure):
    """Mirror of dh_product in include/dethead.h."""
    _fields_ = ([(n, L.c_void_p) for n in ("a", "b", "bias", "residual", "out", "z")]
                + [(n, L.c_i64) for n in ("lda", "ldb", "ldo", "ldr", "a_batch", "b_batch", "o_batch", "res_batch")]
                + [(n, L.c_int) for n in ("I", "J", "R", "batch", "a_by_reduction", "b_by_reduction", "bias_on_i", "reduce_batch")])


def _address(t):
    return t.data_ptr() if t is not None else 0


def _run(products, dtype, activation, device):
    """One launch of the given products: dicts of tensors and geometry (see dh_product)."""
    n = len(products)
    table = (Product * n)(*[Product(**p) for p in products])
    lib = L.lib()
    code = _DTYPES[dtype]
    need = lib.dh_products_workspace(table, n, code)
    ws = L.workspace(need, device) if need else None
    with L.device_guard(device):
        L.check(lib.dh_products(table, n, code, activation, L.ptr(ws), need, L.stream()), "dh_products")


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
        L.check(lib.dh_product_slope(L.ptr(dy), L.ptr(z), L.ptr(dz), L.ptr(dbias), outer, n, inner, activation, _DTYPES[dy.dtype],
                                     L.ptr(ws), need, L.stream()), "dh_product_slope")
    return dz, dbias


# ---- geometry: rows (M, K) -> (M, N) and maps (B, K, P) -> (B, N, P), both with the weight (N, K) ----

def _rows_forward(x, w, bias, residual, out, z):
    m, k = x.shape
    return dict(a=_address(x), b=_address(w), bias=_address(bias), residual=_address(residual), out=_address(out), z=_address(z),
                lda=x.stride(0), ldb=k, ldo=out.stride(0), ldr=residual.stride(0) if residual is not None else 0,
                I=m, J=w.shape[0], R=k, batch=1, a_by_reduction=1, b_by_reduction=1)


def _rows_grad_input(dz, w, out):
    return dict(a=_address(dz), b=_address(w), out=_address(out), lda=dz.shape[1], ldb=w.shape[1], ldo=w.shape[1],
                I=dz.shape[0], J=w.shape[1], R=dz.shape[1], batch=1, a_by_reduction=1, b_by_reduction=0)


def _rows_grad_weight(dz, x, out):
    return dict(a=_address(dz), b=_address(x), out=_address(out), lda=dz.shape[1], ldb=x.stride(0), ldo=x.shape[1],
                I=dz.shape[1], J=x.shape[1], R=x.shape[0], batch=1, a_by_reduction=0, b_by_reduction=0)


def _maps_forward(x, w, bias, residual, out, z):
    b, k, p = x.shape
    n = w.shape[0]
    return dict(a=_address(w), b=_address(x), bias=_address(bias), residual=_address(residual), out=_address(out), z=_address(z),
                lda=k, ldb=p, ldo=p, ldr=p, b_batch=x.stride(0), o_batch=n * p,
                res_batch=residual.stride(0) if residual is not None else 0,
                I=n, J=p, R=k, batch=b, a_by_reduction=1, b_by_reduction=0, bias_on_i=1)


def _maps_grad_input(dz, w, out):
    b, n, p = dz.shape
    k = w.shape[1]
    return dict(a=_address(w), b=_address(dz), out=_address(out), lda=k, ldb=p, ldo=p, b_batch=n * p, o_batch=k * p,
                I=k, J=p, R=n, batch=b, a_by_reduction=0, b_by_reduction=0)


def _maps_grad_weight(dz, x, out):
    b, n, p = dz.shape
    k = x.shape[1]
    return dict(a=_address(dz), b=_address(x), out=_address(out), lda=p, ldb=p, ldo=k, a_batch=n * p, b_batch=x.stride(0),
                I=n, J=k, R=p, batch=b, a_by_reduction=1, b_by_reduction=1, reduce_batch=1)


def _forward(rows, act, items, want_z):
    """items: (x, w, bias, residual) with x (M, K) or (B, K, P) -> outputs, pre-activations."""
    make = _rows_forward if rows else _maps_forward
    x = items[0][0]
    shape = (lambda x, w: (x.shape[0], w.shape[0])) if rows else (lambda x, w: (x.shape[0], w.shape[0], x.shape[2]))
    outs = [torch.empty(shape(x, w), dtype=x.dtype, device=x.device) for x, w, _, _ in items]
    zs = [torch.empty_like(o) if want_z else None for o in outs]
    _run([make(x, w, b, r, o, z) for (x, w, b, r), o, z in zip(items, outs, zs)], x.dtype, act, x.device)
    return outs, zs


class _Products(torch.autograd.Function):
    """The products of one launch with their gradients.  tensors: x, w, bias, residual of each (bias, residual may be None)."""

    @staticmethod
    def forward(ctx, rows, act, *tensors):
        items = [tensors[k:k + 4] for k in range(0, len(tensors), 4)]
        outs, zs = _forward(rows, act, items, act != 0)
        ctx.rows, ctx.act, ctx.n = rows, act, len(items)
        ctx.save_for_backward(*[t for (x, w, _, _), z in zip(items, zs) for t in (x, w, z)])
        return tuple(outs)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        rows, saved, wants = ctx.rows, ctx.saved_tensors, ctx.needs_input_grad
        result, inputs, weights = [None, None], [], []
        for k in range(ctx.n):
            x, w, z = saved[3 * k:3 * k + 3]
            want_x, want_w, want_b, want_r = wants[2 + 4 * k:6 + 4 * k]
            dy = grads[k]
            dx = dw = db = None
            if dy is None:
                result += [None] * 4
                continue
            dy = dy.contiguous()
            if want_x or want_w or want_b:
                outer, n, inner = (dy.shape[0], dy.shape[1], 1) if rows else dy.shape
                dz, db = _slope(dy, z, ctx.act, want_b, outer, n, inner)
                if want_x:
                    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
                    inputs.append((_rows_grad_input if rows else _maps_grad_input)(dz, w, dx) | {"keep": dz})
                if want_w:
                    dw = torch.empty(w.shape, dtype=w.dtype, device=w.device)
                    weights.append((_rows_grad_weight if rows else _maps_grad_weight)(dz, x, dw) | {"keep": dz})
            result += [dx, dw, db, dy if want_r else None]
        keep = [p.pop("keep") for p in inputs + weights]
        device = saved[0].device
        for group in (inputs, weights):
            if group:
                _run(group, saved[0].dtype, 0, device)
        del keep
        return tuple(result)


def _apply(rows, act, items):
    tensors = [t for item in items for t in item]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return list(_Products.apply(rows, act, *tensors))
    return _forward(rows, act, items, False)[0]


def _activation(name, where):
    if name not in ACTIVATIONS:
        raise ValueError(f"{where}: activation must be one of {list(ACTIVATIONS)}, got {name!r}")
    return ACTIVATIONS[name]


def _checked(where, x, weight, bias, residual):
    """The tensors in one supported type on one ROCm device (cast to autocast's type where that is on)."""
    tensors = [x, weight, bias, residual]
    for t, name in zip(tensors, ("x", "weight", "bias", "residual")):
        if t is None and name in ("bias", "residual"):
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{where}: {name} must be a torch.Tensor, got {type(t).__name__}")
        if not t.is_cuda:
            raise RuntimeError(f"{where}: {name} is on {t.device}: object_detection_amd only runs on ROCm devices (no CPU fallback)")
        if t.device != x.device:
            raise RuntimeError(f"{where}: {name} is on {t.device}, x on {x.device}")
    if torch.is_autocast_enabled("cuda"):
        dtype = torch.get_autocast_dtype("cuda")
        tensors = [t.to(dtype) if t is not None and t.is_floating_point() else t for t in tensors]
    for t, name in zip(tensors, ("x", "weight", "bias", "residual")):
        if t is not None and (t.dtype != tensors[0].dtype or t.dtype not in _DTYPES):
            raise RuntimeError(f"{where}: x, weight, bias and residual must have one type, fp32, fp16 or bf16; {name} is {t.dtype}, "
                               f"x {tensors[0].dtype}")
    return tensors


def _check_weight(where, weight, bias, inputs):
    if weight.dim() not in (2, 4) or (weight.dim() == 4 and weight.shape[2:] != (1, 1)) or weight.shape[1] != inputs:
        raise RuntimeError(f"{where}: weight must be (outputs, {inputs}) or (outputs, {inputs}, 1, 1), got {tuple(weight.shape)}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise RuntimeError(f"{where}: bias must be ({weight.shape[0]},), got {tuple(bias.shape)}")


def _as_rows(t):
    """(..., C) -> (M, C) with the last axis dense and one stride between rows; a copy only where the strides do not allow a
    view (or rows overlap, as in an expanded tensor)."""
    t = t.reshape(t.shape[:-1].numel(), t.shape[-1]) if t.dim() != 2 else t
    if t.shape[-1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t


def linear(x, weight, bias=None, activation=None, residual=None):
    """act(x weight^T + bias) + residual for x (..., C), weight (N, C), bias (N,), residual (..., N) -> (..., N).

    activation: None, "relu", "silu", "gelu" (the exact one, with erf) or "sigmoid".  From one row to many; rows of x and of the
    residual may be strided (a slice of a wider tensor is read in place)."""
    act = _activation(activation, "linear")
    x, weight, bias, residual = _checked("linear", x, weight, bias, residual)
    if x.dim() < 1 or weight.dim() != 2:
        raise RuntimeError(f"linear: x must be (..., C) and weight (N, C), got {tuple(x.shape)} and {tuple(weight.shape)}")
    _check_weight("linear", weight, bias, x.shape[-1])
    shape = x.shape[:-1] + weight.shape[:1]
    if residual is not None:
        if residual.shape != shape:
            raise RuntimeError(f"linear: residual must be {tuple(shape)}, got {tuple(residual.shape)}")
        residual = _as_rows(residual)
    out, = _apply(True, act, [(_as_rows(x), weight.contiguous(), bias.contiguous() if bias is not None else None, residual)])
    return out.view(shape)


def _planes(t):
    """(B, C, ny, nx) -> (B, C, P) with dense planes; images may be apart (a slice of a wider tensor)."""
    b, c, h, w = t.shape
    if t.stride()[1:] == (h * w, w, 1) and t.stride(0) >= c * h * w:
        return t.view(b, c, h * w) if t.is_contiguous() else t.as_strided((b, c, h * w), (t.stride(0), h * w, 1))
    return t.contiguous().view(b, c, h * w)


def _channels_last(t):
    return t.dim() == 4 and t.is_contiguous(memory_format=torch.channels_last) and not t.is_contiguous()


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
    weight = weight.reshape(n, c).contiguous()
    bias = bias.contiguous() if bias is not None else None
    if _channels_last(x):
        rows = x.permute(0, 2, 3, 1).reshape(-1, c)
        res = _as_rows(residual.permute(0, 2, 3, 1).reshape(-1, n)) if residual is not None else None
        out, = _apply(True, act, [(rows, weight, bias, res)])
        return out.view(b, h, w, n).permute(0, 3, 1, 2)
    out, = _apply(False, act, [(_dense(x), weight, bias, _dense(residual) if residual is not None else None)])
    return out.view(b, n, h, w)


def _dense(t):
    """_planes() through autograd: torch's own view operations where a gradient has to find its way back."""
    if t.requires_grad and torch.is_grad_enabled():
        b, c, h, w = t.shape
        return t.reshape(b, c, h * w) if t.is_contiguous() else t.contiguous().view(b, c, h * w)
    return _planes(t)


def head_convs(xs, weights, biases):
    """The 1x1 convolutions of a detection head, all levels in one launch (yolo.py:52): xs[l] (B, C_l, ny_l, nx_l), weights[l]
    (N, C_l, 1, 1) or (N, C_l), biases[l] (N,) or None -> the list of (B, N, ny_l, nx_l).  At most five levels."""
    xs, weights, biases = list(xs), list(weights), list(biases)
    if not xs or len(xs) > MAX_PRODUCTS or len(weights) != len(xs) or len(biases) != len(xs):
        raise RuntimeError(f"head_convs: 1 to {MAX_PRODUCTS} levels with a weight and a bias each, got {len(xs)}, {len(weights)}, {len(biases)}")
    items, shapes = [], []
    for l, (x, weight, bias) in enumerate(zip(xs, weights, biases)):
        x, weight, bias, _ = _checked(f"head_convs, level {l}", x, weight, bias, None)
        if x.dim() != 4:
            raise RuntimeError(f"head_convs, level {l}: x must be (B, C, ny, nx), got {tuple(x.shape)}")
        _check_weight(f"head_convs, level {l}", weight, bias, x.shape[1])
        if items and (x.dtype != items[0][0].dtype or x.device != items[0][0].device):
            raise RuntimeError(f"head_convs, level {l}: {x.dtype} on {x.device}, level 0 {items[0][0].dtype} on {items[0][0].device}")
        items.append((_dense(x), weight.reshape(weight.shape[0], -1).contiguous(), bias.contiguous() if bias is not None else None, None))
        shapes.append((x.shape[0], weight.shape[0]) + tuple(x.shape[2:]))
    return [o.view(s) for o, s in zip(_apply(False, 0, items), shapes)]
