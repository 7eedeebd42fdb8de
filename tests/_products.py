"""The products of object_detection_amd.layers in 64 bits, with bounds on how far a kernel may be from them.

Bounds count roundings, u = 2^-24 for fp32 and half a step of the type T for what is stored in it:
  * z = sum_r a b + bias: at most (R + 1) roundings of partial sums whose magnitudes stay below S = sum |a b| + |bias|, so
    |dz| <= (R + 2) u S (one more for a residual bias addition); products of 16-bit values are exact in fp32;
  * y = act(z) + residual: the slope of every activation is at most 1.13, so 1.13 |dz|, plus the function's own error: at most
    8 u (1 + |z|) (an exp or erf of 2 ulp and three operations), plus one rounding of the addition, plus the rounding to T;
  * a gradient at z is dy * act'(z'), z' being z as stored in T: |act''| <= 0.8, so 0.8 |dy| (|z| uT + |dz|) + 8 u |dy| (1 + |z|),
    plus the rounding of the product to T where it enters a product (not where it is summed for the bias);
  * the products of the backward propagate those bounds through |W| and |x| and add their own (R + 2) u sum and rounding."""
import torch

U32 = 2.0 ** -24
LOWEST = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}      # half the smallest step


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def act64(z, name):
    """act, act'."""
    if name is None:
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).double()
    if name == "sigmoid":
        s = torch.sigmoid(z)
        return s, s * (1 - s)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    normal = torch.special.ndtr(z)
    return z * normal, normal + z * torch.exp(-z * z / 2) * 0.3989422804014327


def rows64(x, w, bias, act, residual, dy=None):
    """Values and bounds of one product over rows; x (M, K), w (N, K), on the device the tensors are on.  Returns {name: (value,
    bound)}."""
    dtype = x.dtype
    ut, low = half_step(dtype), LOWEST[dtype]
    X, W = x.double(), w.double()
    k = X.shape[1]
    z = X @ W.t()
    size = X.abs() @ W.abs().t()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    ez = (k + 2) * U32 * size
    y, slope = act64(z, act)
    ey = ez if act is None else 1.13 * ez + 8 * U32 * (1 + z.abs())
    if residual is not None:
        y = y + residual.double()
        ey = ey + U32 * y.abs()
    out = {"y": (y, ey + ut * (y.abs() + ey) + low)}
    if dy is None:
        return out
    G = dy.double()
    dz = G * slope
    if act is None:
        esum = eop = torch.zeros_like(dz)
    elif act == "relu":
        esum, eop = torch.zeros_like(dz), torch.zeros_like(dz)       # (callers keep z away from 0)
    else:
        esum = G.abs() * (0.8 * (z.abs() * ut + ez + low) + 8 * U32 * (1 + z.abs()))
        eop = esum + ut * (dz.abs() + esum) + low
    m, n = dz.shape
    dx, ex = dz @ W, eop @ W.abs() + (n + 2) * U32 * ((dz.abs() + eop) @ W.abs())
    dw, ew = dz.t() @ X, eop.t() @ X.abs() + (m + 2) * U32 * ((dz.abs() + eop).t() @ X.abs())
    db, eb = dz.sum(0), esum.sum(0) + (m + 2) * U32 * (dz.abs() + esum).sum(0)
    for name, v, e in (("dx", dx, ex), ("dw", dw, ew), ("db", db, eb)):
        out[name] = (v, e + ut * (v.abs() + e) + low)
    out["dr"] = (G, torch.zeros_like(G))
    return out


def close(got, want, label=""):
    value, bound = want
    got = got.detach().to(value.device).double().reshape(value.shape)
    off = (got - value).abs()
    bad = ~(off <= bound)
    if bad.any():
        at = int((off - bound).argmax())
        raise AssertionError(f"{label}: {int(bad.sum())} of {bad.numel()} values out of bounds; worst {off.reshape(-1)[at]:.3e} against "
                             f"{bound.reshape(-1)[at]:.3e} at value {value.reshape(-1)[at]:.6e}")


def to_rows(t):
    """(B, C, ny, nx) -> (B * ny * nx, C)."""
    return t.permute(0, 2, 3, 1).reshape(-1, t.shape[1])


def to_maps(rows, like):
    b, _, h, w = like.shape
    return rows.reshape(b, h, w, -1).permute(0, 3, 1, 2)
