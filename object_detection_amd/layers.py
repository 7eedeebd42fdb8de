"""Matrix products with bias, activation and residual in one launch: the 1x1 convolutions of the detection head
(object_detection/yolov5/models/yolo.py:41,52) and of the blocks before it, on channel-major maps, and the same operator on rows.

  y = act(W x + b) + residual

Sums, bias, activation and residual are fp32 and the result is rounded once.  All three entries are differentiable (x, weight,
bias, residual) and take fp32, fp16 or bf16 tensors of one type; under torch.autocast their inputs are cast to its type, as
torch's own layers do.  The backward of an activation reads the pre-activation, kept in the tensors' type.  A second derivative is
not offered.
"""
import ctypes

from . import _lib as L

MAX_LEVELS = 5          # of head_convs(): DH_MAX_PRODUCTS of include/dethead.h
ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "sigmoid": 4}


class Product(ctypes.Structure):
    """Mirror of dh_product in include/dethead.h."""
    _fields_ = ([(n, L.c_void_p) for n in ("a", "b", "bias", "residual", "out", "z", "a_sum")]
                + [(n, L.c_i64) for n in ("lda", "ldb", "ldo", "ldr", "a_batch", "b_batch", "o_batch", "res_batch")]
                + [(n, L.c_int) for n in ("I", "J", "R", "batch", "a_by_reduction", "b_by_reduction", "bias_on_i", "reduce_batch")])


def _activation(name, where):
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"{where}: activation must be one of {list(ACTIVATIONS)}, got {name!r}") from None


def linear(x, weight, bias=None, activation=None, residual=None):
    """act(x weight^T + bias) + residual for x (..., C), weight (N, C), bias (N,), residual (..., N) -> (..., N).

    activation: None, "relu", "silu", "gelu" (the exact one, with erf) or "sigmoid".  From one row to many; rows of x and of the
    residual may be strided (a slice of a wider tensor is read in place)."""
    return L.host().linear(x, weight, bias, _activation(activation, "linear"), residual)


def pointwise_conv(x, weight, bias=None, activation=None, residual=None):
    """A 1x1 convolution with its epilogue: act(conv(x) + bias) + residual for x (B, C, ny, nx), weight (N, C) or (N, C, 1, 1),
    bias (N,), residual (B, N, ny, nx) -> (B, N, ny, nx).

    activation as in linear().  A channels_last x runs as rows and gives a channels_last result."""
    return L.host().pointwise_conv(x, weight, bias, _activation(activation, "pointwise_conv"), residual)


def head_convs(xs, weights, biases):
    """The 1x1 convolutions of a detection head, all levels in one launch (yolo.py:52): xs[l] (B, C_l, ny_l, nx_l), weights[l]
    (N, C_l, 1, 1) or (N, C_l), biases[l] (N,) or None -> the list of (B, N, ny_l, nx_l).  At most five levels."""
    return L.host().head_convs(xs, weights, biases)
