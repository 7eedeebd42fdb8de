"""Products with bias, activation and residual in the epilogue, and their gradients, against 64 bits (tests/_products.py)."""
import ctypes

import pytest
import torch

from tests._products import LOWEST, close, rows64, to_maps, to_rows

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = [None, "relu", "silu", "gelu", "sigmoid"]


def made(shape, dtype, seed, factor=1.0, whole=False):
    """Seeded values; `whole`: small integers, whose products and sums are exact (a relu's border is then exactly zero)."""
    g = torch.Generator().manual_seed(seed)
    if whole:
        return torch.randint(-3, 4, shape, generator=g).to(dtype)
    return (torch.randn(shape, generator=g) * factor).to(dtype)


def rows_case(m, k, n, dtype, act, bias, residual, seed=0):
    whole = act == "relu"
    x = made((m, k), dtype, seed, whole=whole)
    w = made((n, k), dtype, seed + 1, max(k, 1) ** -0.5, whole=whole)
    b = made((n,), dtype, seed + 2, 0.5, whole=whole) if bias else None
    r = made((m, n), dtype, seed + 3) if residual else None
    dy = made((m, n), dtype, seed + 4)
    return x, w, b, r, dy


def leaves(*tensors):
    return [t.cuda().requires_grad_(True) if t is not None else None for t in tensors]


def check_rows(m, k, n, dtype, act, bias, residual):
    from object_detection_amd.layers import linear
    x, w, b, r, dy = rows_case(m, k, n, dtype, act, bias, residual)
    want = rows64(x, w, b, act, r, dy)
    label = f"rows {m}x{k}->{n} {dtype} {act}"
    with torch.no_grad():
        y = linear(x.cuda(), w.cuda(), b.cuda() if bias else None, act, r.cuda() if residual else None)
    assert y.shape == (m, n) and y.dtype == dtype
    close(y, want["y"], label + " y")
    gx, gw, gb, gr = leaves(x, w, b, r)
    y2 = linear(gx, gw, gb, act, gr)
    assert torch.equal(y2.detach(), y)                      # the same arithmetic with and without a backward to come
    y2.backward(dy.cuda())
    close(gx.grad, want["dx"], label + " dx")
    close(gw.grad, want["dw"], label + " dw")
    if bias:
        close(gb.grad, want["db"], label + " db")
    if residual:
        assert torch.equal(gr.grad.cpu(), dy)


SIZES = [(1, 1, 1), (1, 64, 64), (3, 5, 7), (2, 8, 264), (17, 129, 65), (64, 64, 64), (128, 64, 128), (130, 200, 257), (65, 1000, 33),
         (7, 2049, 12), (200, 24, 8), (513, 72, 136)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_rows_sizes(size, dtype):
    check_rows(*size, dtype, "silu", True, True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True), (True, True)])
def test_rows_epilogues(act, dtype, bias, residual):
    check_rows(37, 72, 88, dtype, act, bias, residual)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(4096, 256, 512), (1, 4096, 1024), (9, 4096, 777), (2000, 40, 40)])
def test_rows_larger(size, dtype):
    check_rows(*size, dtype, "gelu", True, False)


MAPS = [(1, 1, 1, 1, 1), (2, 16, 255, 5, 7), (1, 130, 65, 13, 13), (3, 64, 64, 8, 8), (2, 33, 130, 20, 20), (5, 8, 24, 1, 3),
        (1, 512, 255, 4, 4), (2, 128, 255, 40, 40), (70, 16, 16, 2, 2)]


def check_maps(b, k, n, ny, nx, dtype, act, residual, layout=torch.contiguous_format):
    from object_detection_amd.layers import pointwise_conv
    whole = act == "relu"
    x = made((b, k, ny, nx), dtype, 1, whole=whole).contiguous(memory_format=layout)
    w = made((n, k, 1, 1), dtype, 2, k ** -0.5, whole=whole)
    bias = made((n,), dtype, 3, 0.5, whole=whole)
    r = made((b, n, ny, nx), dtype, 4) if residual else None
    dy = made((b, n, ny, nx), dtype, 5)
    want = rows64(to_rows(x), w.reshape(n, k), bias, act, to_rows(r) if residual else None, to_rows(dy))
    label = f"maps {b}x{k}x{ny}x{nx}->{n} {dtype} {act} {layout}"
    gx, gw, gb, gr = leaves(x, w, bias, r)
    y = pointwise_conv(gx, gw, gb, act, gr)
    assert y.shape == (b, n, ny, nx) and y.dtype == dtype
    close(to_rows(y), want["y"], label + " y")
    y.backward(dy.cuda())
    close(to_rows(gx.grad), want["dx"], label + " dx")
    close(gw.grad.reshape(n, k), want["dw"], label + " dw")
    close(gb.grad, want["db"], label + " db")
    if residual:
        assert torch.equal(gr.grad.cpu(), dy)
    return y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", MAPS)
def test_maps_sizes(size, dtype):
    check_maps(*size, dtype, "silu", True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_maps_activations(act, dtype):
    check_maps(2, 40, 48, 6, 6, dtype, act, False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_maps_channels_last(dtype):
    y = check_maps(2, 40, 72, 5, 6, dtype, "silu", True, torch.channels_last)
    assert y.is_contiguous(memory_format=torch.channels_last)


# Sizes that reach every tile shape (128 x 128 in both step lengths, 256 x 256, the thin kernel's one and two row blocks, split
# reductions of each), with edges that fill no tile; the 64-bit side runs on the GPU.
LARGE = [(4100, 136, 1040, "silu", True), (4100, 1048, 1040, "gelu", False), (8200, 520, 4080, None, True), (16, 4096, 2056, "silu", True),
         (17, 2056, 2100, "gelu", True), (32, 520, 4096, None, False), (5, 1001, 2049, "silu", True), (700, 8192, 72, "silu", True),
         (3001, 333, 1501, "silu", True), (1000, 333, 1001, "silu", True), (333, 1001, 1000, None, False), (700, 100, 900, "gelu", True)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n,act,residual", LARGE)
def test_rows_every_shape(m, k, n, act, residual, dtype):
    from object_detection_amd.layers import linear
    x, w, b, r, dy = [t.cuda() for t in rows_case(m, k, n, dtype, act, True, True, seed=3)]
    r = r if residual else None
    want = rows64(x, w, b, act, r, dy)
    gx, gw, gb = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = linear(gx, gw, gb, act, r)
    close(y, want["y"], "y")
    y.backward(dy)
    close(gx.grad, want["dx"], "dx")
    close(gw.grad, want["dw"], "dw")
    close(gb.grad, want["db"], "db")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,k,n,ny,nx,act", [(8, 128, 255, 80, 80, None), (6, 72, 250, 52, 52, "silu"), (4, 512, 512, 52, 64, None),
                                             (3, 100, 260, 75, 61, "gelu"), (130, 40, 264, 13, 13, "silu")])
def test_maps_every_shape(b, k, n, ny, nx, act, dtype):
    from object_detection_amd.layers import pointwise_conv
    x, w, bias = made((b, k, ny, nx), dtype, 1).cuda(), made((n, k, 1, 1), dtype, 2, k ** -0.5).cuda(), made((n,), dtype, 3, 0.5).cuda()
    r, dy = made((b, n, ny, nx), dtype, 4).cuda(), made((b, n, ny, nx), dtype, 5).cuda()
    want = rows64(to_rows(x), w.reshape(n, k), bias, act, to_rows(r), to_rows(dy))
    gx, gw, gb = [t.clone().requires_grad_(True) for t in (x, w, bias)]
    y = pointwise_conv(gx, gw, gb, act, r)
    close(to_rows(y), want["y"], "y")
    y.backward(dy)
    close(to_rows(gx.grad), want["dx"], "dx")
    close(gw.grad.reshape(n, k), want["dw"], "dw")
    close(gb.grad, want["db"], "db")


@pytest.mark.parametrize("dtype", DTYPES)
def test_head_levels(dtype):
    """Three levels of different widths and sizes in one launch; one level without a bias."""
    from object_detection_amd.layers import head_convs
    geometry = [(16, 12, 12), (40, 6, 6), (129, 3, 3)]
    xs = [made((3, c, h, w), dtype, 10 + c) for c, h, w in geometry]
    ws = [made((75, c, 1, 1), dtype, 20 + c, c ** -0.5) for c, _, _ in geometry]
    bs = [made((75,), dtype, 30), None, made((75,), dtype, 31)]
    dys = [made((3, 75, h, w), dtype, 40 + h) for _, h, w in geometry]
    gx, gw, gb = leaves(*xs), leaves(*ws), leaves(*bs)
    ys = head_convs(gx, gw, gb)
    torch.autograd.backward(ys, [d.cuda() for d in dys])
    for l in range(3):
        want = rows64(to_rows(xs[l]), ws[l].reshape(75, -1), bs[l], None, None, to_rows(dys[l]))
        assert ys[l].shape == dys[l].shape
        close(to_rows(ys[l]), want["y"], f"level {l} y")
        close(to_rows(gx[l].grad), want["dx"], f"level {l} dx")
        close(gw[l].grad.reshape(75, -1), want["dw"], f"level {l} dw")
        if bs[l] is not None:
            close(gb[l].grad, want["db"], f"level {l} db")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_rows_inside_a_wider_tensor(dtype, offset):
    """x and the residual as column slices of tensors whose other columns are NaN: nothing around a row is read into it."""
    from object_detection_amd.layers import linear
    x, w, b, r, dy = rows_case(70, 40, 56, dtype, "silu", True, True)
    wide = torch.full((70, 40 + offset + 9), float("nan"), dtype=dtype, device="cuda")
    wide_r = torch.full((70, 56 + offset + 8), float("nan"), dtype=dtype, device="cuda")
    wide[:, offset:offset + 40] = x.cuda()
    wide_r[:, offset:offset + 56] = r.cuda()
    gx, gr = wide[:, offset:offset + 40].detach().requires_grad_(True), wide_r[:, offset:offset + 56].detach().requires_grad_(True)
    assert not gx.is_contiguous()
    gw, gb = leaves(w, b)
    y = linear(gx, gw, gb, "silu", gr)
    want = rows64(x, w, b, "silu", r, dy)
    close(y, want["y"], "y")
    y.backward(dy.cuda())
    close(gx.grad, want["dx"], "dx")
    close(gw.grad, want["dw"], "dw")


@pytest.mark.parametrize("dtype", DTYPES)
def test_maps_inside_a_wider_tensor(dtype):
    """Channels of a wider map (a concatenation's slice), its other channels NaN; odd cells, so nothing is aligned."""
    from object_detection_amd.layers import pointwise_conv
    x, w = made((3, 20, 5, 5), dtype, 1), made((17, 20), dtype, 2, 0.2)
    wide = torch.full((3, 27, 5, 5), float("nan"), dtype=dtype, device="cuda")
    wide[:, 3:23] = x.cuda()
    with torch.no_grad():
        y = pointwise_conv(wide[:, 3:23], w.cuda())
    close(to_rows(y), rows64(to_rows(x), w, None, None, None)["y"], "y")


def test_broadcast_residual_and_gradient():
    """An expanded residual and an expanded output gradient (sum()) are read and differentiated as what they stand for."""
    from object_detection_amd.layers import linear
    x, w, b, _, _ = rows_case(24, 16, 40, torch.float32, "silu", True, False)
    row = made((1, 40), torch.float32, 9)
    gx, gw, gb, grow = leaves(x, w, b, row)
    linear(gx, gw, gb, "silu", grow.expand(24, 40)).sum().backward()
    want = rows64(x, w, b, "silu", row.expand(24, 40), torch.ones(24, 40))
    close(gx.grad, want["dx"], "dx")
    close(gw.grad, want["dw"], "dw")
    close(gb.grad, want["db"], "db")
    assert torch.equal(grow.grad.cpu(), torch.full((1, 40), 24.0))


def test_the_same_tensor_twice():
    """x as its own residual (y = act(x W^T) + x): its gradient is the sum of both paths."""
    from object_detection_amd.layers import linear
    x, w, b, _, dy = rows_case(19, 48, 48, torch.float32, "silu", True, False)
    gx, gw = leaves(x, w)
    y = linear(gx, gw, b.cuda(), "silu", gx)
    y.backward(dy.cuda())
    want = rows64(x, w, b, "silu", x, dy)
    close(y, want["y"], "y")
    value, bound = want["dx"]
    close(gx.grad, (value + dy.double(), bound + 2 * 2.0 ** -24 * (value.abs() + dy.abs())), "dx")


@pytest.mark.parametrize("size", [(0, 8, 8), (5, 0, 9), (5, 8, 0), (0, 0, 3)])
def test_empty(size):
    from object_detection_amd.layers import linear
    m, k, n = size
    x, w, b, r, dy = rows_case(m, k, n, torch.float32, "silu", True, True)
    want = rows64(x, w, b, "silu", r, dy)
    gx, gw, gb, gr = leaves(x, w, b, r)
    y = linear(gx, gw, gb, "silu", gr)
    assert y.shape == (m, n)
    close(y, want["y"], "y")
    y.backward(dy.cuda())
    for g, name in ((gx, "dx"), (gw, "dw"), (gb, "db")):
        close(g.grad, want[name], name)


def test_infinities_and_nan_stay_in_their_rows():
    """An infinite or NaN input reaches its own output row only, as in the definition."""
    from object_detection_amd.layers import linear
    for dtype in DTYPES:
        x, w, b, _, _ = rows_case(140, 72, 130, dtype, None, True, False)
        want = rows64(x, w, b, None, None)["y"]
        x[7, 3], x[20, 71], x[139, 0] = float("nan"), float("inf"), float("-inf")
        with torch.no_grad():
            y = linear(x.cuda(), w.cuda(), b.cuda()).cpu()
        special = [7, 20, 139]
        exact = x.double()[special] @ w.double().t() + b.double()
        assert torch.equal(torch.isnan(y[special]), torch.isnan(exact))
        finite = ~torch.isnan(exact)
        assert torch.equal(y[special].double()[finite], exact[finite])
        rest = torch.ones(140, dtype=torch.bool)
        rest[special] = False
        close(y[rest], (want[0][rest], want[1][rest]), f"rest {dtype}")


@pytest.mark.parametrize("small,large", [(1e-36, 1e6), (1e-30, 1e-6), (3e38, 1e-20), (2.0 ** -100, 1.0), (0.0, 1.0)])
@pytest.mark.parametrize("size", [(70, 200, 90), (600, 96, 9000)])
def test_fp32_over_its_whole_range(size, small, large):
    """fp32 products of values near both ends of the range keep fp32's accuracy (their parts may leave bf16's, see the kernel)."""
    from object_detection_amd.layers import linear
    m, k, n = size
    g = torch.Generator().manual_seed(9)
    x = ((torch.rand((m, k), generator=g) + 0.1) / 1.1).mul_(small).cuda()
    w = ((torch.rand((n, k), generator=g) - 0.5)).mul_(large).cuda()
    with torch.no_grad():
        y = linear(x, w)
    close(y, rows64(x, w, None, None, None)["y"], "y")
    mixed = x.clone()
    mixed[:, ::3] = 0.0
    mixed[5, 7] = 1e-38                     # one subnormal-to-be among ordinary values and zeros
    with torch.no_grad():
        y = linear(mixed, w)
    close(y, rows64(mixed, w, None, None, None)["y"], "with zeros")


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_activations_far_out(act):
    """Pre-activations from -1e4 to 1e4: no overflow on the way, the limits of the functions at the ends."""
    from object_detection_amd.layers import linear
    z = torch.tensor([-1e4, -200.0, -100.0, -88.0, -20.0, -5.0, -1.0, -0.0, 0.0, 1.0, 5.0, 20.0, 88.0, 100.0, 200.0, 1e4])
    x, w = z[:, None], torch.ones(1, 1)
    want = rows64(x, w, None, act, None, torch.ones(16, 1))
    gx = x.cuda().requires_grad_(True)
    y = linear(gx, w.cuda(), activation=act)
    y.sum().backward()
    close(y, want["y"], "y")
    close(gx.grad, want["dx"], "dx")


def test_gradient_against_differences():
    """The directional derivative of <dy, y> by central differences of the kernel itself (fp32): step h = 2^-6 has an error of
    h^2/6 of the third derivative (|act'''| < 1.1 over the direction's projections, below 2e-4 of the terms' sum) and the
    rounding of y, 2 (R + 4) u sum |dy| (|y| + 1) / h."""
    from object_detection_amd.layers import linear
    m, k, n, h = 12, 24, 20, 2.0 ** -6
    for act in ("silu", "gelu", "sigmoid"):
        x, w, b, r, dy = rows_case(m, k, n, torch.float32, act, True, True, seed=5)
        vx, vw, vb = made((m, k), torch.float32, 50, 0.3), made((n, k), torch.float32, 51, 0.3 * k ** -0.5), made((n,), torch.float32, 52, 0.3)
        t = [v.cuda() for v in (x, w, b, r, dy, vx, vw, vb)]

        def value(s):
            with torch.no_grad():
                y = linear(t[0] + s * t[5], t[1] + s * t[6], t[2] + s * t[7], act, t[3])
            return (y.double() * t[4].double()).sum()
        gx, gw, gb = leaves(x, w, b)
        linear(gx, gw, gb, act, t[3]).backward(t[4])
        slope = sum((g.grad.double() * v.double()).sum() for g, v in ((gx, t[5]), (gw, t[6]), (gb, t[7])))
        got = (value(h) - value(-h)) / (2 * h)
        y = linear(*t[:3], act, t[3]).double()
        # direction of z: (x + s vx)(w + s vw)^T is quadratic in s, its first and second derivatives bound the third of act(z(s))
        z1 = (t[5] @ t[1].t() + t[0] @ t[6].t() + t[7]).double().abs()
        z2 = 2 * (t[5] @ t[6].t()).double().abs()
        third = 1.1 * z1 ** 3 + 3 * 0.8 * z1 * z2
        bound = (t[4].double().abs() * (h * h / 6 * 1.5 * third + 2 * (k + 4) * 2.0 ** -24 * (y.abs() + 1) / h)).sum()
        assert (got - slope).abs() < bound, (act, float(got), float(slope), float(bound))


@pytest.mark.parametrize("which", [0, 1, 2, 3, (0, 3), (1, 2), (2, 3)])
@pytest.mark.parametrize("act", [None, "silu"])
def test_gradients_of_some_inputs_only(which, act):
    """Each of x, weight, bias and residual alone, and pairs of them: the wanted gradients and no others."""
    from object_detection_amd.layers import head_convs, linear
    which = which if isinstance(which, tuple) else (which,)
    x, w, b, r, dy = rows_case(33, 40, 24, torch.float32, act, True, True)
    want = rows64(x, w, b, act, r, dy)
    t = [v.cuda().requires_grad_(k in which) for k, v in enumerate((x, w, b, r))]
    linear(t[0], t[1], t[2], act, t[3]).backward(dy.cuda())
    for k, name in enumerate(("dx", "dw", "db", "dr")):
        if k in which:
            close(t[k].grad, want[name], name)
        else:
            assert t[k].grad is None
    # levels without a bias between levels with one, only some of them trained
    xs = [x.view(1, 33, 40, 1).permute(0, 2, 1, 3).cuda() for _ in range(3)]
    ws, bs = [w.cuda().requires_grad_(l != 1) for l in range(3)], [b.cuda().requires_grad_(True), None, b.cuda().requires_grad_(True)]
    ys = head_convs(xs, ws, bs)
    (ys[0].sum() + 2 * ys[2].sum()).backward()          # level 1 takes no part
    one = rows64(x, w, b, None, None, torch.ones(33, 24))
    two = rows64(x, w, b, None, None, torch.full((33, 24), 2.0))
    close(ws[0].grad, one["dw"], "level 0")
    close(ws[2].grad, two["dw"], "level 2")
    close(bs[0].grad, one["db"], "level 0 bias")
    close(bs[2].grad, two["db"], "level 2 bias")
    assert ws[1].grad is None


def test_saved_inputs_are_guarded():
    """An input that is overwritten between forward and backward is an error, not a wrong gradient."""
    from object_detection_amd.layers import linear
    x, w, _, _, _ = rows_case(8, 16, 8, torch.float32, None, False, False)
    gx, gw = x.cuda(), w.cuda().requires_grad_(True)
    y = linear(gx, gw)
    gx.zero_()
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_autocast_casts_like_torch_layers():
    from object_detection_amd.layers import head_convs, linear
    x, w, b, _, _ = rows_case(9, 32, 24, torch.float32, None, True, False)
    gx, gw, gb = leaves(x, w, b)
    with torch.autocast("cuda", dtype=torch.float16):
        y = linear(gx, gw, gb)
        maps = head_convs([gx.view(1, 9, 32, 1).permute(0, 2, 1, 3)], [gw], [gb])[0]
    assert y.dtype == torch.float16 and maps.dtype == torch.float16
    y.float().sum().backward()
    assert gx.grad.dtype == gw.grad.dtype == torch.float32
    h = rows64(x.half(), w.half(), b.half(), None, None, torch.ones(9, 24, dtype=torch.float16))
    close(y, h["y"], "y")
    close(gx.grad, h["dx"], "dx")
    close(maps.permute(0, 2, 3, 1).reshape(9, 24), h["y"], "maps")


def test_same_bits_every_time():
    """Split reductions are joined in a fixed order: outputs and gradients repeat bit for bit."""
    from object_detection_amd.layers import linear
    x, w, b, r, dy = rows_case(2000, 300, 40, torch.bfloat16, "silu", True, True)
    runs = []
    for _ in range(3):
        gx, gw, gb = leaves(x, w, b)
        y = linear(gx, gw, gb, "silu", r.cuda())
        y.backward(dy.cuda())
        runs.append([y.detach(), gx.grad, gw.grad, gb.grad])
    for again in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], again))


def test_another_stream_and_graph_replay():
    """The calls run on torch's current stream; captured into a graph (forward and gradients) they replay on new inputs."""
    from object_detection_amd.layers import linear
    x, w, b, r, dy = [t.cuda() for t in rows_case(50, 640, 72, torch.float16, "silu", True, True)]
    side = torch.cuda.Stream()
    with torch.no_grad():
        eager = linear(x, w, b, "silu", r)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = linear(x, w, b, "silu", r)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(eager, other)
    sx, sdy = x.clone().requires_grad_(True), dy.clone()
    gw = w.clone().requires_grad_(True)

    def step():
        y = linear(sx, gw, b, "silu", r)
        return (y.detach(),) + torch.autograd.grad(y, [sx, gw], sdy)
    with torch.cuda.stream(side):
        for _ in range(2):
            out = step()
    torch.cuda.synchronize()
    del out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (70, 71, 72):
        fresh = made((50, 640), torch.float16, seed).cuda()
        with torch.no_grad():
            sx.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = step()
        torch.cuda.synchronize()
        for a, c in zip(got, want):
            assert torch.equal(a, c)
        del want


def test_entry_leaves_everything_around_the_output():
    """dh_products into the middle of a larger buffer: rows, columns and batches around the output keep their bits."""
    from object_detection_amd import _lib as L
    from object_detection_amd.layers import Product
    for dtype, code in ((torch.float32, 0), (torch.bfloat16, 2)):
        for i, j, k, ldo in ((5, 7, 33, 12), (130, 129, 64, 136), (64, 64, 640, 64)):
            a, b = made((i, k), dtype, 1).cuda(), made((j, k), dtype, 2).cuda()
            frame = torch.full((i + 4, ldo), 77.0, dtype=dtype, device="cuda")
            p = (Product * 1)(Product(a=a.data_ptr(), b=b.data_ptr(), out=frame[2].data_ptr(), lda=k, ldb=k, ldo=ldo, I=i, J=j, R=k,
                                      batch=1, a_by_reduction=1, b_by_reduction=1))
            need = L.lib().dh_products_workspace(p, 1, code)
            ws = torch.full((need + 64,), 7, dtype=torch.uint8, device="cuda")
            assert L.lib().dh_products(p, 1, code, 0, ctypes.c_void_p(ws.data_ptr()), need, L.stream()) == 0
            torch.cuda.synchronize()
            close(frame[2:2 + i, :j], rows64(a.cpu(), b.cpu(), None, None, None)["y"], f"{dtype} {i}x{j}")
            keep = frame.clone()
            keep[2:2 + i, :j] = 77.0
            assert (keep == 77.0).all() and (ws[need:] == 7).all()


def test_refuses_what_it_cannot_do():
    from object_detection_amd.layers import head_convs, linear, pointwise_conv
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(6, 8, device="cuda")
    for call in (lambda: linear(x, w.half()), lambda: linear(x.double(), w.double()), lambda: linear(x, w[:, :7]),
                 lambda: linear(x, w, torch.zeros(5, device="cuda")), lambda: linear(x, w, residual=torch.zeros(4, 5, device="cuda")),
                 lambda: linear(x, w.cpu()), lambda: linear(x, torch.zeros(6, 8, 1, 1, device="cuda")),
                 lambda: pointwise_conv(x, w), lambda: pointwise_conv(x.view(1, 8, 2, 2), torch.zeros(6, 8, 3, 3, device="cuda")),
                 lambda: pointwise_conv(x.view(1, 8, 2, 2), w, residual=torch.zeros(1, 6, 2, 3, device="cuda")),
                 lambda: head_convs([], [], []), lambda: head_convs([x.view(1, 8, 2, 2)] * 6, [w] * 6, [None] * 6),
                 lambda: head_convs([x.view(1, 8, 2, 2)], [w, w], [None]), lambda: linear(x.to_sparse(), w), lambda: linear(x.long(), w.long()),
                 lambda: head_convs([x.view(1, 8, 2, 2), x.half().view(1, 8, 2, 2)], [w, w.half()], [None, None])):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        linear(x, w, activation="softmax")
    y = linear(x.requires_grad_(True), w, activation="silu")
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_views_with_the_sign_beside_them():
    """The imaginary part of a conjugate is a view of the memory of its negative: as input, weight, bias, residual and gradient."""
    from object_detection_amd.layers import linear
    c = torch.tensor([[2.0 + 3.0j]], device="cuda")
    v = c.conj().imag
    assert v.is_neg() and float(v) == -3.0
    one, two = torch.ones(1, 1, device="cuda"), torch.full((1, 1), 2.0, device="cuda")
    assert float(linear(v, two)) == -6.0
    assert float(linear(two, v)) == -6.0
    assert float(linear(two, one, v[0], None, v)) == -4.0
    x = two.clone().requires_grad_(True)
    y = linear(x, two)
    (dx,) = torch.autograd.grad(y, x, v)
    assert float(dx) == -6.0


@pytest.mark.parametrize("m,k,n", [(200, 512, 190), (130, 1024, 64), (64, 96, 4096)])
def test_values_that_underflow_among_others(m, k, n):
    """Values below 2^-100 here and there, in whole rows of x, in whole columns of the weight, rows of zeros: every element to fp32's
    own error, k roundings of the sum of its products' magnitudes (and k halves of the smallest step)."""
    from object_detection_amd.layers import linear
    g = torch.Generator().manual_seed(13)
    x, w, dy = (torch.randn(*s, generator=g) for s in ((m, k), (n, k), (m, n)))
    few = torch.rand(m, k, generator=g) < 0.02
    x[few] *= 2.0 ** -torch.randint(100, 140, (int(few.sum()),), generator=g).float()
    dy[torch.rand(m, n, generator=g) < 0.02] *= 2.0 ** -118
    for scenario in range(6):
        if scenario == 1: x[5] = torch.randn(k, generator=g) * 2.0 ** -120
        if scenario == 2: x[m - 1] = 2.0 ** -70 * torch.randn(k, generator=g) * 2.0 ** -62
        if scenario == 3: x[7] = 0.0
        if scenario == 4: w[3] *= 2.0 ** -119
        if scenario == 5: dy[:, 2] = dy[:, 2].sign() * 2.0 ** -121
        gx, gw, gb = leaves(x, w, torch.zeros(n))
        y = linear(gx, gw, gb)
        y.backward(dy.cuda())
        x64, w64, dy64 = x.double(), w.double(), dy.double()
        for got, a, b, terms in ((y, x64, w64.t(), k), (gx.grad, dy64, w64, n), (gw.grad, dy64.t(), x64, m), (gb.grad, dy64.t(), torch.ones(m, 1).double(), m)):
            want, size = a @ b, a.abs() @ b.abs()
            off = (got.detach().cpu().double().reshape(want.shape) - want).abs()
            assert bool((off <= (terms + 2) * (size * 2.0 ** -24 + 2.0 ** -150)).all()), (scenario, float((off / size.clamp_min(1e-300)).max()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k", [8, 64, 72, 128, 192, 200, 256, 320, 1016, 1024, 1032, 4096])
def test_reductions_shorter_and_longer_than_the_ring(dtype, k):
    """One step and less to many of them, whole and partial last ones, on few tiles, in all three products."""
    check_rows(72, k, 136, dtype, "silu", True, True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(1, 4096, 1024), (32, 2048, 80), (32, 2049, 80), (32, 2048, 1), (16, 4096, 16), (17, 4096, 16),
                                   (1, 1, 1), (32, 1000, 777), (1, 65536, 3), (2, 65536, 3)])
def test_few_rows_and_few_outputs(dtype, m, k, n):
    """Either side of where a few rows stop being worked on straight from memory."""
    check_rows(m, k, n, dtype, "sigmoid", True, False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(33, 512, 512), (64, 1024, 16), (65, 1023, 17), (127, 40, 100), (128, 1, 1), (129, 7, 260), (256, 512, 1024),
                                   (257, 1024, 816), (300, 96, 800), (1024, 1024, 256), (1025, 1024, 240), (4097, 33, 48), (64, 1025, 64)])
def test_short_products_of_some_rows(dtype, m, k, n):
    """Groups of 64 rows, whole and partial, either side of where tiles take over."""
    check_rows(m, k, n, dtype, "silu", True, True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("b,ny,nx", [(2, 0, 5), (2, 5, 0), (0, 4, 5), (0, 0, 0), (3, 0, 1)])
def test_maps_without_cells(b, ny, nx, act, dtype):
    """No images, or images without cells: zero gradients for what is trained, all of it together and each alone."""
    from object_detection_amd.layers import head_convs, pointwise_conv
    for trained in ((0, 1, 2, 3), (0,), (1,), (2,), (1, 2)):
        t = [made((b, 8, ny, nx), dtype, 1), made((16, 8, 1, 1), dtype, 2), made((16,), dtype, 3), made((b, 16, ny, nx), dtype, 4)]
        t = [v.cuda().requires_grad_(k in trained) for k, v in enumerate(t)]
        y = pointwise_conv(t[0], t[1], t[2], act, t[3])
        assert y.shape == (b, 16, ny, nx)
        y.sum().backward()
        for k in trained:
            assert t[k].grad.shape == t[k].shape and not t[k].grad.any()
    x, w, bias = made((b, 8, ny, nx), dtype, 1).cuda(), made((16, 8), dtype, 2).cuda(), made((16,), dtype, 3).cuda().requires_grad_(True)
    head_convs([x, x], [w, w], [bias, bias])[1].sum().backward()
    assert not bias.grad.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_slope_entry_without_elements_writes_zeros(dtype):
    """dbias of no elements is zero; the buffers beside it, here with room, are neither read (they hold NaN) nor written."""
    from object_detection_amd import _lib as L
    code = DTYPES.index(dtype)
    n, guard = 40, torch.full((4096,), float("nan"), dtype=dtype, device="cuda")
    ws = torch.full((L.lib().dh_product_slope_workspace(n),), 255, dtype=torch.uint8, device="cuda")
    for outer, inner in ((3, 0), (0, 1), (0, 9), (0, 0)):
        for z in (None, guard.data_ptr()):
            dbias = torch.full((n + 8,), 5.0, dtype=dtype, device="cuda")
            dz = torch.full((4096,), 3.0, dtype=dtype, device="cuda")
            assert L.lib().dh_product_slope(guard.data_ptr(), z, dz.data_ptr(), dbias.data_ptr(), outer, n, inner, 2, code, ws.data_ptr(), ws.numel(),
                                            L.stream()) == 0
            torch.cuda.synchronize()
            assert not dbias[:n].any() and (dbias[n:] == 5).all() and (dz == 3).all()


@pytest.mark.parametrize("m,k,n", [(200, 512, 190), (600, 96, 9000), (70, 200, 90), (520, 640, 1040)])
@pytest.mark.parametrize("small,large", [(2.0 ** -140, 2.0 ** 100), (2.0 ** -149, 2.0 ** 120), (2.0 ** -134, 1.0), (2.0 ** -133, 2.0 ** 20)])
def test_an_operand_of_nothing_but_the_smallest_values(m, k, n, small, large):
    """All of x, or of the output's gradient, subnormal: their first bf16 part is zero, the products are not.  The bound is fp32's: k
    roundings of the sum of the magnitudes, and halves of the smallest step.  The bias gradient adds at most 600 equal magnitudes of at
    most 2^17 smallest steps, which fp32 does without an error."""
    from object_detection_amd.layers import linear
    g = torch.Generator().manual_seed(17)
    sign = lambda *s: torch.randint(0, 2, s, generator=g).float() * 2 - 1
    x, w, dy = sign(m, k) * small, (torch.rand(n, k, generator=g) + 0.5) * large, sign(m, n) * small
    x[:, ::5] = 0.0
    gx, gw, gb = leaves(x, w, torch.zeros(n))
    with torch.no_grad():
        y = linear(gx, gw)
    X, W, D = x.double().cuda(), w.double().cuda(), dy.double().cuda()

    def hold(got, a, b, terms, label):
        want, size = a @ b, a.abs() @ b.abs()
        bound = (terms + 2) * (size * 2.0 ** -24 + 2.0 ** -150)
        assert bool(((got.double().reshape(want.shape) - want).abs() <= bound).all()), label
        assert float(want.abs().max()) > 2 * float(bound.max()), label                       # (zeros would not pass)
    hold(y, X, W.t(), k, "y")
    linear(gx, gw, gb).backward(dy.cuda())
    hold(gx.grad, D, W, n, "dx")
    assert torch.equal(gb.grad.double(), D.sum(0))
    # the weight's gradient needs the other operand large
    big = ((torch.rand(m, k, generator=g) + 0.5) * large).cuda()
    gw2 = w.cuda().requires_grad_(True)
    linear(big, gw2).backward(dy.cuda())
    hold(gw2.grad, D.t(), big.double(), m, "dw")


@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("trained", [(0,), (1,), (2,), (0, 1, 2, 3)])
@pytest.mark.parametrize("layout", ["contiguous", "copied"])
def test_second_derivatives_are_refused(layout, trained, act):
    """Through the gradient of each input, also where a copy of the input was read and where nothing else is trained: an error, not a
    term left out."""
    from object_detection_amd.layers import head_convs, linear, pointwise_conv
    def inputs(*shapes):
        t = [made(s, torch.float32, 60 + k).cuda() for k, s in enumerate(shapes)]
        if layout == "copied":
            t = [v.transpose(0, 1).contiguous().transpose(0, 1) if v.dim() > 1 else torch.stack([v, v], 1)[:, 0] for v in t]
        return [v.requires_grad_(k in trained) for k, v in enumerate(t)]
    calls = ((linear, inputs((6, 8), (10, 8), (10,), (6, 10))), (pointwise_conv, inputs((2, 8, 3, 4), (10, 8), (10,), (2, 10, 3, 4))))
    for call, (x, w, b, r) in calls:
        t = [v for k, v in enumerate((x, w, b, r)) if k in trained]
        y = call(x, w, b, act, r)
        grads = torch.autograd.grad(y.sum(), t, create_graph=True)
        for k, g in zip(trained, grads):
            if k == 3:                                                  # the residual's gradient is dy itself: constant here
                assert not g.requires_grad
                continue
            with pytest.raises(RuntimeError, match="second derivative"):
                (y.sum() + g.square().sum()).backward(retain_graph=True)
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad(g.sum(), t, retain_graph=True, allow_unused=True)
    x, w, b, _ = calls[1][1]
    if trained != (0, 1, 2, 3):
        ys = head_convs([x, x.detach()], [w, w.detach()], [b, b.detach()])
        t = (x, w, b)[trained[0]]
        g, = torch.autograd.grad(ys[0].sum() + ys[1].sum(), t, create_graph=True)
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(g.sum(), t)


def test_a_gradient_of_a_residual_can_be_differentiated():
    """dr = dy, so what dy depends on can be reached through it; and first derivatives under create_graph are the ordinary ones."""
    from object_detection_amd.layers import linear
    x, w, b, r, dy = rows_case(7, 16, 12, torch.float32, "silu", True, True)
    gx, gw, gb, gr, gdy = leaves(x, w, b, r, dy)
    y = linear(gx, gw, gb, "silu", gr)
    dr, dx, dw, db = torch.autograd.grad(y, (gr, gx, gw, gb), gdy, create_graph=True)
    want = rows64(x, w, b, "silu", r, dy)
    for got, name in ((dx, "dx"), (dw, "dw"), (db, "db")):
        close(got, want[name], name)
    back, = torch.autograd.grad((dr * dr).sum(), gdy, retain_graph=True)
    assert torch.equal(back, 2 * gdy.detach())
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(dx.sum(), gdy)


@pytest.mark.parametrize("trained", [False, True])
def test_forward_mode_is_refused(trained):
    """A dual input, weight, bias or residual: an error, not a result without its tangent.  Where forward mode is off, or the level has
    ended, the calls run."""
    import torch.autograd.forward_ad as ad
    from object_detection_amd.grads import clip_grads, total_grad_norm
    from object_detection_amd.layers import head_convs, linear, pointwise_conv
    t = [made(s, torch.float32, 80 + k).cuda().requires_grad_(trained) for k, s in enumerate(((1, 8, 4, 5), (6, 8, 1, 1), (6,), (1, 6, 4, 5)))]
    rows = [made(s, torch.float32, 90 + k).cuda().requires_grad_(trained) for k, s in enumerate(((20, 8), (6, 8), (6,), (20, 6)))]
    with ad.dual_level():
        for k in range(4):
            dual = [ad.make_dual(v, torch.ones_like(v)) if e == k else v for e, v in enumerate(t)]
            dual_rows = [ad.make_dual(v, torch.ones_like(v)) if e == k else v for e, v in enumerate(rows)]
            calls = [lambda: pointwise_conv(*dual[:3], "silu", dual[3]), lambda: linear(*dual_rows[:3], "silu", dual_rows[3])]
            if k < 3:
                calls.append(lambda: head_convs([t[0], dual[0]], [t[1], dual[1]], [t[2], dual[2]]))
            for call in calls:
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
                with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
                    call()
                with ad._set_fwd_grad_enabled(False):
                    call()
        g = ad.make_dual(torch.ones(5, device="cuda"), torch.ones(5, device="cuda"))
        for call in (lambda: total_grad_norm([g]), lambda: clip_grads([g], 1.0)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
    pointwise_conv(*t[:3], "silu", t[3])


def test_forward_mode_of_a_fused_head_is_refused():
    import torch.autograd.forward_ad as ad
    from object_detection_amd.yolo import Detect
    det = Detect(3, [[1, 2, 3, 4]], (8,)).cuda().train()
    x = torch.randn(1, 8, 5, 6, device="cuda")
    det.fused_convs = True
    with ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        det([ad.make_dual(x, torch.ones_like(x))])
    assert det([x])[0].shape == (1, 2, 5, 6, 8)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
def test_16_bit_activations_relative_to_their_own_size(act, dtype):
    """Far out an activation and its slope are small numbers that 16 bits still hold: each to 2^-13 of its terms' magnitudes (the
    approximations' 2^-14, and arguments up to 126 whose roundings an exponential multiplies, 126 * 2^-24), fp32's own 2^-22 where
    terms near 1 cancel, one rounding to the type, and what underflows in fp32 (|z| 2^-125)."""
    from object_detection_amd.layers import linear
    g = torch.Generator().manual_seed(3)
    z = torch.cat([torch.linspace(-16, 16, 1501), torch.linspace(-100, 100, 401), torch.rand(2000, generator=g) * 12 - 12]).to(dtype)
    n = z.numel()
    for rows, wide in ((n, 1), (1, n)):                     # z = x w with either of them 1: exact
        x, w = (z[:, None], torch.ones(1, 1, dtype=dtype)) if wide == 1 else (torch.ones(1, 1, dtype=dtype), z[:, None])
        gx = x.cuda().requires_grad_(wide == 1)
        y = linear(gx, w.cuda(), activation=act)
        Z = z.double().reshape(rows, wide)
        s, tail = torch.special.expit(Z), torch.special.expit(-Z)
        normal, bell = torch.erfc(-Z * 0.5 ** 0.5) / 2, torch.exp(-Z * Z / 2) * 0.3989422804014327        # (ndtr ends at 1e-16)
        value = {"silu": Z * s, "gelu": Z * normal, "sigmoid": s}[act]
        low = LOWEST[dtype]
        close(y, (value, value.abs() * (2.0 ** -13 + torch.finfo(dtype).eps / 2 * 1.001) + low + Z.abs() * 2.0 ** -125 + 2.0 ** -126), f"{act} value")
        if wide == 1:
            y.sum().backward()
            slope = {"silu": s * (1 + Z * tail), "gelu": normal + Z * bell, "sigmoid": s * tail}[act]
            terms = {"silu": s * (1 + Z.abs() * (tail + 2.0 ** -9)), "gelu": normal + Z.abs() * bell, "sigmoid": s * tail + s * 2.0 ** -9}[act]
            close(gx.grad, (slope, terms * 2.0 ** -13 + slope.abs() * torch.finfo(dtype).eps / 2 * 1.001 + low + (1 + Z.abs()) * 2.0 ** -125),
                  f"{act} slope")


def test_a_fused_head_takes_what_its_layers_take():
    """Six levels, doubles, levels of different types, a patched layer and a module-wide hook: the layers' own results; the ordinary head
    is one launch."""
    from object_detection_amd import yolo
    from object_detection_amd.yolo import Detect

    def head(nl, dtype=torch.float32):
        det = Detect(3, [[1, 2, 3, 4]] * nl, (8,) * nl).to(device="cuda", dtype=dtype).train()
        det.fused_convs = True
        det.lazy_maps = True
        return det, [made((2, 8, 5 + l, 6), dtype, l).cuda() for l in range(nl)]
    launches = []
    real = yolo.head_convs
    yolo.head_convs = lambda *a: launches.append(1) or real(*a)
    try:
        def run(det, xs, fused):
            del launches[:]
            got = det._convolutions(list(xs))
            assert len(launches) == fused
            for g, m, x in zip(got, det.m, xs):
                want = m(x)
                assert g.dtype == want.dtype and g.shape == want.shape
                if not fused:
                    assert torch.equal(g, want)
        for nl, fused in ((1, 1), (3, 1), (5, 1), (6, 0)):
            run(*head(nl), fused)
        run(*head(3, torch.float64), 0)
        det, xs = head(3)
        det.m[1].double()
        run(det, [xs[0], xs[1].double(), xs[2]], 0)
        det, xs = head(2)
        det.m[1].half()
        run(det, [xs[0], xs[1].half()], 0)
        det, xs = head(2)
        plain = det.m[0].forward
        det.m[0].forward = lambda x: plain(x) + 1
        run(det, xs, 0)
        del det.m[0].forward
        run(det, xs, 1)
        seen = []
        handle = torch.nn.modules.module.register_module_forward_hook(lambda m, *a: seen.append(m))
        try:
            run(det, xs, 0)
        finally:
            handle.remove()
        assert det.m[0] in seen and det.m[1] in seen
        with torch.autocast("cuda", dtype=torch.float16):
            del launches[:]
            got = det._convolutions([xs[0], xs[1].half()])
            assert launches == [1] and all(g.dtype == torch.float16 for g in got)
        with torch.autocast("cuda", dtype=torch.float16), pytest.raises(RuntimeError):      # as its layers do
            det._convolutions([xs[0].double(), xs[1]])
    finally:
        yolo.head_convs = real


class _Given(torch.nn.Module):
    """A level's convolution whose output is already there."""

    def __init__(self, conv, out):
        super().__init__()
        self.weight, self.bias, self.out = conv.weight, conv.bias, out

    def forward(self, x):
        return self.out


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("lazy", [False, True])
def test_a_fused_head_in_eval(lazy, half):
    """The fused convolutions against 64 bits, what follows them bit for bit what an ordinary head makes of the same maps, in forward() and
    in detections(), and the decoded values against the unfused head's: by the mean value theorem they differ by the maps' differences
    times the decode's slopes (2 s stride / 4 of a centre, 32/27 anchor of a size, 1/4 of a score), and by the decode's own roundings, eight
    half steps of each."""
    from object_detection_amd.layers import head_convs
    from object_detection_amd.yolo import Detect
    dtype = torch.float16 if half else torch.float32
    torch.manual_seed(4)
    strides = torch.tensor([8.0, 16.0, 32.0])
    det = Detect(20, [[10, 13, 16, 30, 33, 23], [30, 61, 62, 45, 59, 119], [116, 90, 156, 198, 373, 326]], (16, 32, 64)).cuda()
    det.stride = strides
    det.anchors /= strides.view(-1, 1, 1).cuda()
    det = det.to(dtype).eval()
    det.lazy_maps = lazy
    feats = [torch.randn(3, c, s, s + 2, device="cuda").to(dtype) for c, s in ((16, 24), (32, 12), (64, 6))]
    with torch.no_grad():
        det.fused_convs = False
        z0, maps0 = det(list(feats))
        det.fused_convs = True
        z1, maps1 = det(list(feats))
        rows = det.detections(list(feats), 0.3, 0.5)
        convs = head_convs(feats, [m.weight for m in det.m], [m.bias for m in det.m])
        for f, m, y in zip(feats, det.m, convs):
            close(to_rows(y), rows64(to_rows(f).detach(), m.weight.detach().flatten(1), m.bias.detach(), None, None)["y"], "convolution")
        own = list(det.m)
        det.m = torch.nn.ModuleList([_Given(m, y) for m, y in zip(own, convs)])
        z2, maps2 = det(list(feats))
        given = det.detections(list(feats), 0.3, 0.5)
    assert torch.equal(z1, z2) and z1.dtype == z0.dtype and z1.shape == z0.shape
    assert len(maps1) == 3 and all(torch.equal(a, b) for a, b in zip(maps1, maps2))
    assert len(rows) == len(given) == 3 and sum(len(r) for r in rows) > 20
    assert all(torch.equal(a, b) for a, b in zip(rows, given))
    slopes, apart = [], []
    for l, (a, b) in enumerate(zip(maps0, maps1)):
        slope = torch.full((3, 25), 0.25, dtype=torch.float64, device="cuda")
        slope[:, :2] = 0.5 * float(strides[l])
        slope[:, 2:4] = 32 / 27 * (det.anchors[l].double() * float(strides[l]))
        slopes.append((slope[None, :, None, None, :] * (a.double() - b.double()).abs()).reshape(3, -1, 25))
        apart.append(torch.full_like(slopes[-1], float(strides[l])))
    bound = torch.cat(slopes, 1) + 8 * torch.finfo(dtype).eps / 2 * (torch.cat(apart, 1) + z0.double().abs()) * 2
    assert bool(((z0.double() - z1.double()).abs() <= bound).all())
    assert bool(torch.cat(slopes, 1).max() < 1.0)                       # (the bound says something)


def test_function_transforms_are_refused():
    """torch.func's wrapped tensors have no memory of their own: an error, not a result without the transform."""
    from object_detection_amd.grads import total_grad_norm
    from object_detection_amd.layers import linear
    x, w = made((3, 5, 8), torch.float32, 1).cuda(), made((6, 8), torch.float32, 2).cuda()
    for call in (lambda: torch.func.jvp(lambda v: linear(v, w), (x,), (torch.ones_like(x),)), lambda: torch.func.vmap(lambda v: linear(v, w))(x),
                 lambda: torch.func.grad(lambda v: linear(v, w).sum())(x), lambda: torch.func.vmap(lambda v: total_grad_norm([v]))(x),
                 lambda: torch.func.jvp(lambda v: total_grad_norm([v]), (x,), (torch.ones_like(x),))):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [True, False])
def test_a_relu_stops_what_it_stops(rows, dtype):
    """The gradient of a relu is dy or 0: infinities and NaN in dy go no further where z is not positive, and reach x where it is; a NaN
    in z lets dy through.  As torch's relu, value by value."""
    from object_detection_amd.layers import linear, pointwise_conv
    inf, nan = float("inf"), float("nan")
    z, dy = torch.meshgrid(torch.tensor([-inf, -2.0, -0.0, 0.0, 1e-6, 3.0, inf, nan]), torch.tensor([1.0, -2.0, 0.0, inf, -inf, nan]), indexing="ij")
    z, dy = z.reshape(-1).to(dtype), dy.reshape(-1).to(dtype)
    n = z.numel()
    x = (z[:, None] if rows else z.view(1, 1, 6, 8)).cuda().requires_grad_(True)
    g = (dy[:, None] if rows else dy.view(1, 1, 6, 8)).cuda()
    one, bias = torch.ones(1, 1, dtype=dtype, device="cuda"), torch.zeros(1, dtype=dtype, device="cuda", requires_grad=True)
    y = (linear if rows else pointwise_conv)(x, one, bias, "relu")
    y.backward(g)
    ref = x.detach().clone().requires_grad_(True)
    want = torch.relu(ref)
    want.backward(g)
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.nan_to_num(y), torch.nan_to_num(want))
    assert torch.equal(torch.isnan(x.grad), torch.isnan(ref.grad)) and torch.equal(torch.nan_to_num(x.grad), torch.nan_to_num(ref.grad))
    assert torch.isnan(bias.grad).all()
