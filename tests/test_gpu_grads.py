"""Gradient norm and clipping against 64 bits.

The sums are doubles, so the norm is the exact one rounded to fp32: off by at most 2^-24 (1 + 2^-20) relative.  A clipped value is
g * f with f = fp32(min(1, max / (norm + 1e-6)) / scale), two roundings and the one of its own type: 2 * 2^-24 + uT, plus half the
type's smallest step."""
import math

import pytest
import torch

from tests._products import LOWEST, U32, half_step

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SHAPES = [(1,), (3,), (0,), (255, 128, 1, 1), (255,), (64, 32, 3, 3), (8191,), (8192,), (8193,), (7, 5, 3), (1, 1), (20000,)]


def made(shapes, dtype, seed, factor=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * factor * 10.0 ** (k % 4 - 2)).to(dtype).cuda() for k, s in enumerate(shapes)]


def norm64(grads, p, scale=1.0):
    v = torch.cat([g.detach().cpu().double().reshape(-1) for g in grads]).abs() / scale
    return float(v.max()) if p == math.inf else float(v.pow(p).sum().pow(1.0 / p))


def near(got, want):
    assert got.dtype == torch.float32 and got.dim() == 0
    assert abs(float(got) - want) <= want * U32 * 1.001 + LOWEST[torch.float32], (float(got), want)


def clipped_close(out, grads, norm, limit, scale=1.0):
    factor = min(1.0, limit / (norm + 1e-6)) / scale
    for o, g in zip(out, grads):
        want = g.detach().cpu().double() * factor
        off = (o.detach().cpu().double() - want).abs()
        assert bool((off <= want.abs() * (2 * U32 + half_step(o.dtype)) * 1.001 + LOWEST[o.dtype]).all())


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm(dtype, p):
    from object_detection_amd.grads import total_grad_norm
    grads = made(SHAPES, dtype, 1)
    near(total_grad_norm(grads, p), norm64(grads, p))
    near(total_grad_norm(grads, p, scale=torch.tensor(512.0, device="cuda")), norm64(grads, p, 512.0))
    near(total_grad_norm(grads, p, scale=3.0), norm64(grads, p, 3.0))
    near(total_grad_norm(grads[:1], p), norm64(grads[:1], p))
    near(total_grad_norm([grads[2]], p), 0.0)                                # nothing but an empty tensor


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("part", [0.25, 0.999, 4.0])
def test_clip_in_place(dtype, p, part):
    from object_detection_amd.grads import clip_grad_norm_
    grads = made(SHAPES, dtype, 2)
    norm = norm64(grads, p)
    parameters = []
    for g in grads:
        q = torch.nn.Parameter(torch.zeros_like(g))
        q.grad = g.clone()
        parameters.append(q)
    parameters.insert(3, torch.nn.Parameter(torch.zeros(5, device="cuda")))       # one without a gradient
    versions = [q.grad._version for q in parameters if q.grad is not None]
    near(clip_grad_norm_(iter(parameters), norm * part, p), norm)
    after = [q.grad for q in parameters if q.grad is not None]
    clipped_close(after, grads, norm, norm * part)
    assert all(a._version > v for a, v in zip(after, versions))
    if part > 1:
        assert all(torch.equal(a, g) for a, g in zip(after, grads))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fp32_out", [False, True])
def test_clip_into_other_tensors(dtype, fp32_out):
    from object_detection_amd.grads import clip_grads
    grads = made(SHAPES, dtype, 3, 16.0)
    before = [g.clone() for g in grads]
    norm = norm64(grads, 2.0, 64.0)
    out = [torch.full(g.shape, 9.0, dtype=torch.float32 if fp32_out else dtype, device="cuda") for g in grads]
    n, got = clip_grads(grads, 0.5 * norm, scale=64.0, out=out)
    near(n, norm)
    assert all(a is b for a, b in zip(got, out))
    clipped_close(out, grads, norm, 0.5 * norm, 64.0)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    n, made_out = clip_grads(grads, 1e30, scale=64.0)
    assert all(o.dtype == dtype for o in made_out)
    clipped_close(made_out, grads, norm, 1e30, 64.0)
    if not fp32_out:                                                         # some in place, some not
        mixed = [g if k % 2 else o for k, (g, o) in enumerate(zip(grads, out))]
        clip_grads(grads, 0.5 * norm, scale=64.0, out=mixed)
        clipped_close(mixed, before, norm, 0.5 * norm, 64.0)


def test_many_tensors_of_all_types_in_a_bucket():
    """More tensors than one launch holds, of all three types, at odd offsets in their buffers; what lies between stays."""
    from object_detection_amd.grads import clip_grad_norm_
    sizes = [1 + (37 * k) % 300 for k in range(290)]
    parameters, frames, grads = [], [], []
    for dtype in DTYPES:
        frame = torch.full((sum(sizes) + len(sizes),), 5.0, dtype=dtype, device="cuda")
        frames.append(frame)
        at = 1
        for s, g in zip(sizes, made([(s,) for s in sizes], dtype, 4)):
            frame[at:at + s] = g
            q = torch.nn.Parameter(torch.zeros_like(g))
            q.grad = frame[at:at + s]
            parameters.append(q)
            grads.append(g)
            at += s + 1
    norm = norm64(grads, 2.0)
    near(clip_grad_norm_(parameters, 0.1), norm)
    clipped_close([q.grad for q in parameters], grads, norm, 0.1)
    gaps = torch.cumsum(torch.tensor([s + 1 for s in sizes]), 0)
    for frame in frames:
        assert float(frame[0]) == 5.0 and (frame[gaps[:-1].cuda()] == 5.0).all()


def test_layouts():
    """A channels_last gradient, a transposed one and a slice of a wider tensor are clipped where they are."""
    from object_detection_amd.grads import clip_grads, clip_grad_norm_
    base = made([(8, 6, 3, 3), (12, 7), (10, 20)], torch.float32, 5)
    wide = torch.full((10, 25), 3.0, device="cuda")
    wide[:, 2:22] = base[2]
    views = [base[0].contiguous(memory_format=torch.channels_last), base[1].t().contiguous().t(), wide[:, 2:22]]
    norm = norm64(base, 2.0)
    n, out = clip_grads(views, 0.2)
    near(n, norm)
    clipped_close(out, base, norm, 0.2)
    parameters = [torch.nn.Parameter(torch.zeros_like(b)) for b in base]
    for q, v in zip(parameters, views):
        q.grad = v
    near(clip_grad_norm_(parameters, 0.2), norm)
    clipped_close(views, base, norm, 0.2)
    assert (wide[:, :2] == 3.0).all() and (wide[:, 22:] == 3.0).all()


def test_far_ranges():
    """Squares that leave fp32's range, and the smallest numbers."""
    from object_detection_amd.grads import clip_grads
    for size in (1e30, 1e-30, 1e-42):
        g = [torch.full((1000,), size, device="cuda"), torch.full((24,), -size, device="cuda")]
        n, out = clip_grads(g, 1e-3 if size > 1 else 1.0)
        norm = norm64(g, 2.0)
        near(n, norm)
        clipped_close(out, g, norm, 1e-3 if size > 1 else 1.0)


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_not_finite(p):
    from object_detection_amd.grads import clip_grad_norm_, clip_grads, total_grad_norm
    g = [torch.ones(100, device="cuda"), torch.ones(9000, device="cuda")]
    for bad, check in ((float("inf"), math.isinf), (float("-inf"), math.isinf), (float("nan"), math.isnan)):
        for place in (0, 8999):
            h = [t.clone() for t in g]
            h[1][place] = bad
            assert check(float(total_grad_norm(h, p)))
            n, out = clip_grads(h, 1.0, p)
            assert check(float(n))
            want = 0.0 if math.isinf(bad) else float("nan")                 # max / (inf + 1e-6), and NaN
            ref = torch.tensor(1.0) * want
            assert torch.equal(out[0].cpu(), ref.expand(100)) or (math.isnan(want) and torch.isnan(out[0]).all())
            assert math.isnan(float(out[1][place]))
            q = torch.nn.Parameter(torch.zeros(9000, device="cuda"))
            q.grad = h[1].clone()
            with pytest.raises(RuntimeError, match="not finite"):
                clip_grad_norm_(q, 1.0, p, error_if_nonfinite=True)
            assert torch.equal(torch.nan_to_num(q.grad), torch.nan_to_num(h[1]))      # nothing was scaled


def test_limits():
    from object_detection_amd.grads import clip_grad_norm_, clip_grads, total_grad_norm
    assert float(clip_grad_norm_([], 1.0)) == 0.0 and float(total_grad_norm([])) == 0.0
    assert float(clip_grad_norm_([torch.nn.Parameter(torch.zeros(2, device="cuda"))], 1.0)) == 0.0
    z = torch.zeros(100, device="cuda")
    n, out = clip_grads([z], 0.0)                                           # 0 / 1e-6: zero stays zero
    assert float(n) == 0.0 and torch.equal(out[0], z)
    n, out = clip_grads([z + 2], 0.0)
    assert float(n) == 20.0 and torch.equal(out[0], z)
    n, out = clip_grads([z + 2], math.inf)
    assert torch.equal(out[0], z + 2)


def test_refusals():
    from object_detection_amd.grads import clip_grad_norm_, clip_grads, total_grad_norm
    g = torch.ones(4, device="cuda")
    for call in (lambda: clip_grads([g, g.cpu()], 1.0), lambda: clip_grads([g.double()], 1.0), lambda: clip_grads([], 1.0),
                 lambda: clip_grads([g], 1.0, out=[]), lambda: clip_grads([g], 1.0, out=[torch.ones(5, device="cuda")]),
                 lambda: clip_grads([g], 1.0, out=[g.half()]), lambda: clip_grads([g], 1.0, scale=torch.ones(2, device="cuda")),
                 lambda: clip_grads([g, g], 1.0, out=[g, g]), lambda: clip_grads([g, g + 1], 1.0, out=[g.clone(), g]),
                 lambda: clip_grads([g, g], 1.0, out=[g, g.clone()]), lambda: clip_grads([g, g], 1.0, out=[g.clone(), g]),
                 lambda: total_grad_norm([g.to_sparse()]), lambda: total_grad_norm([torch.ones(3)])):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: clip_grads([g], -1.0), lambda: clip_grads([g], math.nan), lambda: clip_grads([g], 1.0, 3.0), lambda: total_grad_norm([g], 0.0)):
        with pytest.raises(ValueError):
            call()
    q = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    q.grad = g.clone()
    with pytest.raises(RuntimeError, match="twice"):
        clip_grad_norm_([q, q], 1.0)
    assert torch.equal(q.grad, g)


def test_a_rank_without_gradients_takes_part_in_the_exchange(monkeypatch):
    from object_detection_amd import grads as G
    met = []

    def exchange(power, norm_type, group):
        met.append((float(power), norm_type, group))
        return power + 16.0                     # what the other ranks hold
    monkeypatch.setattr(G, "all_reduce_norm_power", exchange)
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    assert float(G.clip_grad_norm_([p], 1.0, group=True)) == 4.0 and met == [(0.0, 2.0, None)]
    assert p.grad is None
    with pytest.raises(RuntimeError, match="at least one parameter"):
        G.clip_grad_norm_([], 1.0, group=True)
    assert float(G.clip_grad_norm_([p], 1.0)) == 0.0 and len(met) == 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_factors_below_the_normal_range(dtype):
    """Norms near the end of fp32's range against a small bound: the factor is below 2^-126, the results are not."""
    from object_detection_amd.grads import clip_grads
    g = (torch.randn(10000, generator=torch.Generator().manual_seed(11)) * 1e36).to(dtype)
    norm, (out,) = clip_grads([g.cuda()], 1e-6, out=[torch.empty(10000, device="cuda")])
    want = g.double() * (1e-6 / (g.double().norm() + 1e-6))
    assert 1e-6 / float(norm) < 2.0 ** -140
    # two roundings (the factor, the product) and the exact one by 2^-64: 2^-24 each, and 2^-150 where a result is subnormal
    torch.testing.assert_close(out.cpu().double(), want, rtol=2.1 * 2.0 ** -24, atol=2.0 ** -149)


def test_overlapping_outputs_are_refused():
    from object_detection_amd.grads import clip_grads
    flat = torch.arange(24, device="cuda", dtype=torch.float32)
    kept, half = flat.clone(), torch.ones(16, device="cuda", dtype=torch.float16)
    a, b = torch.ones(8, device="cuda"), torch.ones(8, device="cuda")
    for grads, out in (([a, b], [flat[0:8], flat[7:15]]),               # two outputs share an element
                       ([flat[0:8], b], [a.clone(), flat[4:12]]),       # an output inside another's gradient
                       ([flat[0:24], b], [torch.zeros(24, device="cuda"), flat[16:24]]),
                       ([flat[0:8]], [flat[1:9]]),                      # an output shifted against its own gradient
                       ([half[0:8]], [half.view(torch.float32)])):      # fp32 written over the fp16 that is read
        with pytest.raises(RuntimeError, match="overlap"):
            clip_grads(grads, 1.0, out=out)
    assert torch.equal(flat, kept)
    # neighbours are apart, and one may be written in place while the next is not
    norm, _ = clip_grads([flat[0:8], flat[8:16]], 1e9, out=[flat[0:8], flat[16:24]])
    assert torch.equal(flat[16:24], kept[8:16]) and torch.equal(flat[0:16], kept[0:16])


def test_views_with_the_sign_beside_them():
    """The imaginary part of a conjugate is a view of the memory of its negative."""
    from object_detection_amd.grads import clip_grad_norm_, clip_grads
    c = torch.tensor([[3.0 + 4.0j]], device="cuda")
    g = c.conj().imag
    assert g.is_neg() and float(g) == -4.0
    norm, (out,) = clip_grads([g], 2.0)
    assert float(norm) == 4.0
    torch.testing.assert_close(out.cpu(), torch.full((1, 1), -2.0), rtol=1e-6, atol=0)      # (2 / (4 + 1e-6) is 2.5e-7 off)
    q = torch.nn.Parameter(torch.zeros(1, 1, device="cuda"))
    q.grad = g
    clip_grad_norm_([q], 2.0)
    torch.testing.assert_close(q.grad.cpu(), torch.full((1, 1), -2.0), rtol=1e-6, atol=0)
    torch.testing.assert_close(c.cpu().imag, torch.full((1, 1), 2.0), rtol=1e-6, atol=0)


def test_streams_and_graph_replay():
    from object_detection_amd.grads import clip_grads
    grads = made(SHAPES, torch.float16, 6)
    out = [torch.zeros(g.shape, device="cuda") for g in grads]
    scale = torch.tensor(2.0, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        clip_grads(grads, 0.5, scale=scale, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm, _ = clip_grads(grads, 0.5, scale=scale, out=out)
    for seed in (7, 8, 9):
        for g, f in zip(grads, made(SHAPES, torch.float16, seed)):
            g.copy_(f)
        scale.fill_(float(seed))
        graph.replay()
        torch.cuda.synchronize()
        got, kept = norm.clone(), [o.clone() for o in out]
        again, outs = clip_grads(grads, 0.5, scale=scale, out=[torch.zeros_like(o) for o in out])
        assert torch.equal(got, again) and all(torch.equal(a, b) for a, b in zip(kept, outs))
        near(got, norm64(grads, 2.0, float(seed)))


def test_large_list():
    """More chunks than workgroups, one tensor past 2^25 elements."""
    from object_detection_amd.grads import clip_grads
    g = torch.Generator(device="cuda").manual_seed(1)
    grads = [torch.randn(n, generator=g, device="cuda", dtype=torch.float32) for n in ((1 << 25) + 13, 1 << 20, 77)]
    want = math.sqrt(sum(float(t.double().square().sum()) for t in grads))
    n, out = clip_grads(grads, 10.0)
    near(n, want)
    f = 10.0 / (want + 1e-6)
    for t, o in zip(grads, out):
        assert float((o.double() - t.double() * f).abs().max()) <= float(t.abs().max()) * f * 3 * U32 * 1.001


@pytest.mark.parametrize("count", [176, 177, 280, 281, 600])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lists_around_what_a_launch_takes(dtype, count):
    """Tables that are just full, and several of them; empty tensors at their ends; whole and partial last chunks."""
    from object_detection_amd.grads import clip_grads, total_grad_norm
    sizes = [(0,) if k % 88 in (0, 87) else ((k * 977) % 9000 + 1,) if k % 7 else (8192 * (k % 3 + 1),) for k in range(count)]
    grads = made(sizes, dtype, 12)
    norm = norm64(grads, 2.0)
    near(total_grad_norm(grads), norm)
    for limit in (norm / 3, norm * 3):
        n, out = clip_grads(grads, limit)
        near(n, norm)
        clipped_close(out, grads, norm, limit)
        n, out = clip_grads(grads, limit, out=[torch.empty(s, device="cuda") for s in sizes])
        near(n, norm)
        clipped_close(out, grads, norm, limit)
        mine = [g.clone() for g in grads]
        n, _ = clip_grads(mine, limit, out=mine)
        near(n, norm)
        clipped_close(mine, grads, norm, limit)
        half = [g.clone() for g in grads]                       # every other tensor in place
        n, out = clip_grads(half, limit, out=[g if k % 2 else torch.empty_like(g) for k, g in enumerate(half)])
        near(n, norm)
        clipped_close(out, grads, norm, limit)


def test_training_step_of_the_head():
    """Detect's convolutions, the loss on their outputs, the gradients back to the weights and their clipping, in one run: against
    torch's convolutions on the same device in fp32 and the clipping formula."""
    from object_detection_amd.grads import clip_grad_norm_
    from object_detection_amd.yolo import Detect
    from oracle import yolo as oy
    from tests._synth import synth_targets
    from tests.test_gpu_yolo_loss import make_loss
    import numpy as np
    torch.manual_seed(0)
    anchors = oy.grid_anchors()
    strides = torch.tensor(oy.YOLOV5S_STRIDES)
    det = Detect(80, (anchors * strides.view(-1, 1, 1)).reshape(3, -1).tolist(), (16, 32, 64)).cuda()
    det.stride = strides
    det.anchors.copy_(anchors)
    crit = make_loss(anchors, 80, dict(oy.HYP_SCRATCH))
    feats = [torch.randn(4, c, s, s, device="cuda") for c, s in ((16, 32), (32, 16), (64, 8))]
    targets = torch.from_numpy(synth_targets(np.random.RandomState(3), 40, 4)).cuda()
    results = {}
    for fused in (False, True):
        for lazy in (False, True):
            det.fused_convs, det.lazy_maps = fused, lazy
            det.train()
            det.zero_grad()
            loss, items = crit([m for m in det([f.clone() for f in feats])], targets)
            loss.backward()
            grads = [q.grad.clone() for q in det.parameters()]
            norm = clip_grad_norm_(det.parameters(), 1.0)
            results[fused, lazy] = (loss.detach(), grads, norm, [q.grad for q in det.parameters()])
            near(norm, norm64(grads, 2.0))
            clipped_close([q.grad for q in det.parameters()], grads, norm64(grads, 2.0), 1.0)
            det.grads = None
    base = results[False, False]
    for key, got in results.items():
        # fp32 sums of at most 64 terms in two orders: outputs within 66 u of the terms' sum, the loss and its gradients within
        # 1e-5 of it as the loss' own tests state; the weights' gradients sum 4096 cells
        torch.testing.assert_close(got[0], base[0], rtol=1e-5, atol=1e-6)
        for a, b in zip(got[1], base[1]):
            assert float((a - b).norm()) <= 1e-4 * float(b.norm()), key
    det.eval()
    with torch.no_grad():
        for half in (False, True):
            net = det.half() if half else det
            xs = [f.half() if half else f for f in feats]
            det.fused_convs = False
            z0, maps0 = net(list(xs))
            d0 = net.detections(list(xs), 0.25)
            det.fused_convs = True
            z1, maps1 = net(list(xs))
            d1 = net.detections(list(xs), 0.25)
            for a, b in zip(maps0, maps1):
                torch.testing.assert_close(a, b, rtol=2e-3 if half else 1e-5, atol=4e-3 if half else 1e-5)
            assert z0.shape == z1.shape and len(d0) == len(d1)


def test_a_rank_without_gradients_of_any_kind_takes_part(monkeypatch):
    """Parameters that the kernels would refuse (double, on the host), and no gradients at all: the exchange the others wait in happens."""
    from object_detection_amd import grads as G
    met = []

    def exchange(power, norm_type, group):
        met.append((float(power), power.is_cuda, norm_type))
        return power + 9.0
    monkeypatch.setattr(G, "all_reduce_norm_power", exchange)
    host, double = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(2, device="cuda", dtype=torch.float64))
    for parameters in ([host], [double], [host, double]):
        assert float(G.clip_grad_norm_(parameters, 1.0, group=True)) == 3.0
        assert float(G.clip_grad_norm_(parameters, 1.0, group=True, error_if_nonfinite=True)) == 3.0
    assert len(met) == 9
    assert float(G.total_grad_norm([], group=True)) == 3.0
    norm, out = G.clip_grads([], 1.0, group=True)
    assert float(norm) == 3.0 and out == []
    assert met == [(0.0, True, 2.0)] * 11
    with pytest.raises(RuntimeError):
        G.clip_grads([], 1.0)


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_a_negative_scale(p):
    """|g / scale| does not depend on the scale's sign, g / scale does."""
    from object_detection_amd.grads import clip_grads, total_grad_norm
    grads = made(SHAPES, torch.float32, 21)
    for scale in (-4.0, torch.tensor([-4.0], device="cuda")):
        norm = norm64(grads, p, 4.0)
        near(total_grad_norm(grads, p, scale=scale), norm)
        for limit in (norm / 2, norm * 2, 1e-38 * norm):
            n, out = clip_grads(grads, limit, p, scale=scale, out=[torch.empty_like(g) for g in grads])
            near(n, norm)
            clipped_close(out, [-g for g in grads], norm, limit, 4.0)


def test_strided_gradients_that_share_memory_are_refused():
    """Twice the same columns, an expanded gradient, columns of a tensor that is in the list itself: refused before anything is written.
    Neighbouring columns are apart."""
    from object_detection_amd.grads import clip_grads, clip_grad_norm_
    wide = torch.arange(60, device="cuda", dtype=torch.float32).view(6, 10)
    kept = wide.clone()
    row = torch.ones(1, 8, device="cuda")

    def parameters(*grads):
        ps = [torch.nn.Parameter(torch.zeros(g.shape, device="cuda")) for g in grads]
        for q, g in zip(ps, grads):
            q.grad = g
        return ps
    for grads, match in (((wide[:, 2:5], wide[:, 2:5]), "twice"), ((wide[:, 2:5], wide[:, 2:4]), "twice"), ((row.expand(4, 8),), "share memory"),
                         ((wide, wide[:, 3:5]), "overlap"), ((wide[:, 0:3], wide[0:2]), "overlap")):
        with pytest.raises(RuntimeError, match=match):
            clip_grad_norm_(parameters(*grads), 1.0)
        with pytest.raises(RuntimeError, match=match):
            clip_grads([torch.ones(g.shape, device="cuda") for g in grads], 1.0, out=list(grads))
    assert torch.equal(wide, kept) and (row == 1).all()
    grads = [wide[:, 0:2], wide[:, 2:5], wide[:, 5:9:2]]
    before = [g.clone() for g in grads]
    norm = norm64(before, 2.0)
    near(clip_grad_norm_(parameters(*grads), 3.0), norm)
    clipped_close(grads, before, norm, 3.0)
    assert torch.equal(wide[:, 9], kept[:, 9]) and torch.equal(wide[:, 6:9:2], kept[:, 6:9:2])
    # read as often as one likes: an expanded gradient counts each of its elements, into other tensors
    n, out = clip_grads([row.expand(4, 8), wide[:, 2:5], wide[:, 2:5]], 1e9)
    near(n, norm64([row.expand(4, 8), wide[:, 2:5], wide[:, 2:5]], 2.0))


def test_the_documented_order_with_a_grad_scaler():
    """scale, backward, unscale_, clip_grad_norm_, step: the weights of a step without a scaler whose gradients were clipped by the formula;
    an overflowed step changes nothing.  And `scale` in a loop of its own: the same weights."""
    from object_detection_amd.grads import clip_grad_norm_, clip_grads
    g = made([(40, 16), (40,)], torch.float32, 30)
    start = [torch.zeros_like(v) for v in g]
    norm = norm64(g, 2.0)

    def loss_of(ps):
        return sum((p * v).sum() for p, v in zip(ps, g))          # its gradients are g
    ps = [torch.nn.Parameter(s.clone()) for s in start]
    optimizer = torch.optim.SGD(ps, lr=1.0)
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0)
    scaler.scale(loss_of(ps)).backward()
    scaler.unscale_(optimizer)
    near(clip_grad_norm_(ps, norm / 4), norm)
    scaler.step(optimizer)
    scaler.update()
    clipped_close([-p for p in ps], g, norm, norm / 4)
    after = [p.detach().clone() for p in ps]
    optimizer.zero_grad()
    scaler.scale(loss_of(ps) * float("inf")).backward()
    scaler.unscale_(optimizer)
    assert not math.isfinite(float(clip_grad_norm_(ps, norm / 4)))
    scaler.step(optimizer)
    scaler.update()
    assert all(torch.equal(p, a) for p, a in zip(ps, after)) and scaler.get_scale() == 512.0
    own = [torch.nn.Parameter(s.clone()) for s in start]
    (loss_of(own) * 1024.0).backward()
    n = clip_grad_norm_(own, norm / 4, scale=1024.0)
    near(n, norm)
    clipped_close([p.grad for p in own], g, norm, norm / 4)


def test_a_scale_on_the_host_can_be_captured():
    """A one-element tensor in host memory is a number: nothing is copied, so the call can be captured."""
    from object_detection_amd.grads import clip_grads, total_grad_norm
    grads = made([(100,), (9000,)], torch.float32, 40)
    scale = torch.tensor([8.0], dtype=torch.float64)
    out = [torch.empty_like(g) for g in grads]
    norm = norm64(grads, 2.0, 8.0)
    near(total_grad_norm(grads, scale=scale), norm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n, _ = clip_grads(grads, norm / 2, scale=scale, out=out)
    for _ in range(3):
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        near(n, norm)
        clipped_close(out, grads, norm, norm / 2, 8.0)
