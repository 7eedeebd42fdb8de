"""The workloads on which the products with an epilogue (linear, pointwise_conv, head_convs) and the gradient clipping are
measured: the cases, their inputs, each operator in its plain form (elementary torch operations in 32 bits) and in 64 bits.

`own` selects what `run` does: False computes the plain form, True calls object_detection_amd."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HEAD_CHANNELS = (128, 256, 512)       # feature channels at strides 8, 16, 32 of the small model
STRIDES = (8, 16, 32)
OUTPUTS = 255                         # 3 anchors x (80 classes + 5)
MOST_WORK = {"flops": 141e9, "bytes": 920e6}     # the largest listed case's


def listed():
    return [
        # the three 1x1 convolutions of the head for one image: latency of a detector that serves frame by frame
        {"name": "head_b1_f16", "op": "head", "bs": 1, "img": 640, "outputs": OUTPUTS, "dtype": "f16", "train": False},
        # the same at the benchmark's batch, in the type of its maps
        {"name": "head_b64_f32", "op": "head", "bs": 64, "img": 640, "outputs": OUTPUTS, "dtype": "f32", "train": False},
        # a training step's head under half precision: outputs, and the gradients of features, weights and biases
        {"name": "head_train_b64_f16", "op": "head", "bs": 64, "img": 640, "outputs": OUTPUTS, "dtype": "f16", "train": True},
        # a 1x1 block of the network at stride 8: folded batch norm, SiLU and the shortcut's addition
        {"name": "conv_shortcut_b64_bf16", "op": "conv", "bs": 64, "c1": 128, "c2": 128, "ny": 80, "nx": 80, "dtype": "bf16",
         "activation": "silu", "residual": True, "train": False},
        # the same kind of block, trained in full precision on maps of odd size (416 pixels, stride 32), odd channel counts
        {"name": "conv_odd_train_f32", "op": "conv", "bs": 32, "c1": 384, "c2": 250, "ny": 13, "nx": 13, "dtype": "f32",
         "activation": "silu", "residual": True, "train": True},
        # one token through a projection: reads the weight, does next to nothing with it
        {"name": "linear_token_bf16", "op": "linear", "rows": 1, "c1": 4096, "c2": 4096, "dtype": "bf16", "activation": "silu",
         "residual": False, "train": False},
        # the widening product of a transformer block over many tokens
        {"name": "linear_wide_bf16", "op": "linear", "rows": 8192, "c1": 1024, "c2": 4096, "dtype": "bf16", "activation": "gelu",
         "residual": False, "train": False},
        # a product with shortcut, trained
        {"name": "linear_train_bf16", "op": "linear", "rows": 8192, "c1": 1024, "c2": 1024, "dtype": "bf16", "activation": "silu",
         "residual": True, "train": True},
        # nothing a multiple of anything
        {"name": "linear_odd_f32", "op": "linear", "rows": 1023, "c1": 777, "c2": 1001, "dtype": "f32", "activation": "relu",
         "residual": True, "train": False},
        # the head's own six gradients, when only the head is trained
        {"name": "clip_head_f32", "op": "clip", "width": 0, "depth": 0, "dtype": "f32", "norm": 2.0, "loss_scale": 1.0,
         "clipped": True, "inplace": False},
        # the small model's gradients from a step with a loss scale, into the optimizer's fp32 buffer
        {"name": "clip_small_f16", "op": "clip", "width": 32, "depth": 3, "dtype": "f16", "norm": 2.0, "loss_scale": 1024.0,
         "clipped": True, "inplace": False},
        # the largest model's gradients in place, on a step whose norm stays below the limit (most steps)
        {"name": "clip_large_bf16", "op": "clip", "width": 80, "depth": 6, "dtype": "bf16", "norm": 2.0, "loss_scale": 1.0,
         "clipped": False, "inplace": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["head", "conv", "conv", "linear", "linear", "clip"])
        dtype = rng.choice(["f32", "f16", "bf16"])
        act = rng.choice(["none", "relu", "silu", "gelu", "sigmoid"])
        if op == "head":
            case = {"op": op, "bs": _log_int(rng, 1, 64), "img": 32 * rng.randint(6, 40), "outputs": 3 * (5 + _log_int(rng, 1, 80)),
                    "dtype": dtype, "train": rng.random() < 0.5}
        elif op == "conv":
            case = {"op": op, "bs": _log_int(rng, 1, 64), "c1": _log_int(rng, 16, 512), "c2": _log_int(rng, 16, 512),
                    "ny": _log_int(rng, 10, 160), "nx": _log_int(rng, 10, 160), "dtype": dtype, "activation": act,
                    "residual": rng.random() < 0.5, "train": act != "relu" and rng.random() < 0.4}
        elif op == "linear":
            case = {"op": op, "rows": _log_int(rng, 1, 8192), "c1": _log_int(rng, 64, 4096), "c2": _log_int(rng, 64, 4096),
                    "dtype": dtype, "activation": act, "residual": rng.random() < 0.5,
                    "train": act != "relu" and rng.random() < 0.4}
        else:
            clipped = rng.random() < 0.6
            case = {"op": op, "width": 4 * rng.randint(2, 20), "depth": rng.randint(1, 6), "dtype": dtype,
                    "norm": rng.choice([1.0, 2.0, 2.0, math.inf]), "loss_scale": rng.choice([1.0, 512.0]) if clipped else 1.0,
                    "clipped": clipped, "inplace": not clipped}
        w = work(case)
        if all(w[k] <= MOST_WORK[k] for k in w):
            return case


def _grad_shapes(case):
    """Parameter shapes of a convolutional network: five stages of doubling width, each a strided 3x3 convolution and `depth`
    bottlenecks, a scale and a shift behind every convolution, and the head's convolutions; width 0 is the head alone."""
    w, shapes, before = case["width"], [], 3
    channels = HEAD_CHANNELS if w == 0 else (4 * w, 8 * w, 16 * w)
    for i in range(5 if w else 0):
        c = w << i
        shapes += [(c, before, 3, 3), (c,), (c,)]
        shapes += [(c // 2, c, 1, 1), (c // 2,), (c // 2,), (c, c // 2, 3, 3), (c,), (c,)] * case["depth"]
        before = c
    for c in channels:
        shapes += [(OUTPUTS, c, 1, 1), (OUTPUTS,)]
    return shapes


def _products(case):
    """(batch, inputs, outputs, positions) of every product of a case; tokens are one product of `rows` positions."""
    if case["op"] == "head":
        return [(case["bs"], c, case["outputs"], (case["img"] // s) ** 2) for c, s in zip(HEAD_CHANNELS, STRIDES)]
    if case["op"] == "conv":
        return [(case["bs"], case["c1"], case["c2"], case["ny"] * case["nx"])]
    return [(1, case["c1"], case["c2"], case["rows"])]


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "clip":
        n = sum(math.prod(s) for s in _grad_shapes(case))
        return {"bytes": n * size + 4 + (n * 4 if case["clipped"] else 0), "flops": 2 * n}
    nbytes = flops = 0
    for b, k, n, p in _products(case):
        x, y, w = b * k * p, b * n * p, n * k + n
        nbytes += size * (x + w + y + (y if case.get("residual") else 0))
        flops += 2 * b * n * k * p
        if case["train"]:             # the gradient at the output in; the gradients of input, weight and bias out
            nbytes += size * (y + x + w)
            flops += 4 * b * n * k * p
    return {"bytes": nbytes, "flops": flops}


def _randn(gen, shape, dtype, factor=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * factor).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "clip":
        shapes = _grad_shapes(case)
        sizes = [math.prod(s) for s in shapes]
        # gradients of very different layers: each tensor has a magnitude of its own, over some four decades
        magnitude = torch.exp(torch.rand(len(sizes), generator=gen, device="cuda") * 9.0 - 11.0)
        flat = torch.randn(sum(sizes), generator=gen, device="cuda")
        flat *= magnitude.repeat_interleave(torch.tensor(sizes, device="cuda"), output_size=sum(sizes))
        flat = (flat * case["loss_scale"]).to(dtype)
        size = flat.double().abs() / case["loss_scale"]
        p = case["norm"]
        norm = float(size.max() if p == math.inf else size.pow(p).sum().pow(1.0 / p))
        state["limit"] = norm * (0.3 if case["clipped"] else 3.0)
        state["bucket"] = flat
        if case["inplace"]:           # gradients that are views of one bucket, as DistributedDataParallel keeps them
            state["parameters"] = []
            for s, g in zip(shapes, flat.split(sizes)):
                q = torch.nn.Parameter(torch.empty(s, dtype=dtype, device="cuda"))
                q.grad = g.view(s)
                state["parameters"].append(q)
        else:                         # gradients of their own, and the optimizer's fp32 buffer with a view for each
            state["grads"] = [g.clone().view(s) for s, g in zip(shapes, flat.split(sizes))]
            state["buffer"] = torch.empty(sum(sizes), dtype=torch.float32, device="cuda")
            state["views"] = [v.view(s) for s, v in zip(shapes, state["buffer"].split(sizes))]
            state["scale"] = torch.full((), case["loss_scale"], device="cuda")
        return state
    state["products"] = []
    for b, k, n, p in _products(case):
        if case["op"] == "linear":
            xs, ys, ws = (p, k), (p, n), (n, k)
        else:
            ny, nx = (case["ny"], case["nx"]) if case["op"] == "conv" else (math.isqrt(p), math.isqrt(p))
            xs, ys, ws = (b, k, ny, nx), (b, n, ny, nx), (n, k, 1, 1)
        one = {"x": _randn(gen, xs, dtype), "weight": _randn(gen, ws, dtype, k ** -0.5), "bias": _randn(gen, (n,), dtype, 0.1),
               "residual": _randn(gen, ys, dtype) if case.get("residual") else None,
               "grad": _randn(gen, ys, dtype, 0.01) if case["train"] else None}
        if case["train"]:
            for name in ("x", "weight", "bias"):
                one[name].requires_grad_(True)
        state["products"].append(one)
    return state


def _activate(z, name):
    """act(z) and its derivative."""
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if name == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
        return s, s * (1 - s)
    if name == "gelu":
        c = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * c, c + z * torch.exp(-0.5 * z * z) * (0.5 / math.pi) ** 0.5
    return z, None


def _plain_product(case, one):
    dtype, act = one["x"].dtype, case.get("activation", "none")
    x, w, bias = one["x"].detach().float(), one["weight"].detach().float(), one["bias"].detach().float()
    rows = case["op"] == "linear"
    if rows:
        z = x @ w.t() + bias
    else:
        x = x.flatten(2)
        w = w.flatten(1)
        z = w @ x + bias[:, None]
    y, slope = _activate(z, act) if case["train"] else (_value(z, act), None)
    if one["residual"] is not None:
        y = y + one["residual"].float().view(y.shape)
    y = y.to(dtype).view(one["x"].shape[:-1] + (y.shape[-1],) if rows else (x.shape[0], y.shape[1]) + one["x"].shape[2:])
    if not case["train"]:
        return [y]
    dz = one["grad"].float()
    dz = dz if rows else dz.flatten(2)
    dz = dz if slope is None else dz * slope
    if rows:
        dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    else:
        dx, dw, db = w.t() @ dz, (dz @ x.transpose(1, 2)).sum(0), dz.sum((0, 2))
    return [y, dx.to(dtype).view(one["x"].shape), dw.to(dtype).view(one["weight"].shape), db.to(dtype)]


def _value(z, act):
    """act(z) alone, for a pass without a backward."""
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _plain_clip(state):
    case = state["case"]
    flat = state["bucket"] if case["inplace"] else torch.cat([g.reshape(-1) for g in state["grads"]])
    g = flat.float()
    if not case["inplace"]:
        g = g / state["scale"]
    if case["norm"] == math.inf:
        norm = g.abs().max()
    elif case["norm"] == 1.0:
        norm = g.abs().sum(dtype=torch.float64).float()
    else:
        norm = g.double().square().sum().sqrt().float()
    g = g * (state["limit"] / (norm + 1e-6)).clamp(max=1.0)
    target = state["bucket"] if case["inplace"] else state["buffer"]
    target.copy_(g)
    return [norm, target]


def _own_products(state):
    from object_detection_amd import layers
    case, products = state["case"], state["products"]
    if case["op"] == "head":
        ys = layers.head_convs([o["x"] for o in products], [o["weight"] for o in products], [o["bias"] for o in products])
    else:
        one, act = products[0], case["activation"]
        call = layers.linear if case["op"] == "linear" else layers.pointwise_conv
        ys = [call(one["x"], one["weight"], one["bias"], activation=None if act == "none" else act, residual=one["residual"])]
    if not case["train"]:
        return ys
    leaves = [o[name] for o in products for name in ("x", "weight", "bias")]
    grads = torch.autograd.grad(ys, leaves, [o["grad"] for o in products])
    return [t for i, y in enumerate(ys) for t in (y, *grads[3 * i:3 * i + 3])]


def _own_clip(state):
    from object_detection_amd import grads
    case = state["case"]
    if case["inplace"]:
        return [grads.clip_grad_norm_(state["parameters"], state["limit"], norm_type=case["norm"]), state["bucket"]]
    norm, _ = grads.clip_grads(state["grads"], state["limit"], norm_type=case["norm"], scale=state["scale"], out=state["views"])
    return [norm, state["buffer"]]


def run(state):
    if state["case"]["op"] == "clip":
        return _own_clip(state) if own else _plain_clip(state)
    if own:
        return _own_products(state)
    return [t for one in state["products"] for t in _plain_product(state["case"], one)]


def exact(case, seed):
    """The outputs of run() in 64 bits, from the definitions; positions and channels are one axis each."""
    state = prepare(case, seed)
    if case["op"] == "clip":
        g = state["bucket"].double() / case["loss_scale"]
        p = case["norm"]
        norm = g.abs().max() if p == math.inf else torch.linalg.vector_norm(g, p)
        factor = min(1.0, state["limit"] / (float(norm) + 1e-6))
        return [norm, g * factor]
    outputs = []
    for one in state["products"]:
        planes = case["op"] != "linear"

        def rows_of(t):
            t = t.detach().double()
            return t.flatten(2).transpose(1, 2).reshape(-1, t.shape[1]) if planes else t

        def back(t, like):
            return t.view(like.shape[0], -1, t.shape[1]).transpose(1, 2).reshape(like.shape[0], t.shape[1], *like.shape[2:]) if planes else t

        x, w = rows_of(one["x"]), one["weight"].detach().double().flatten(1)
        z = torch.addmm(one["bias"].detach().double(), x, w.t())
        act = case.get("activation", "none")
        normal = torch.special.ndtr(z) if act == "gelu" else None
        logistic = torch.special.expit(z) if act in ("silu", "sigmoid") else None
        y = {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, 0.0), "silu": lambda: z * logistic,
             "sigmoid": lambda: logistic, "gelu": lambda: z * normal}[act]()
        if one["residual"] is not None:
            y = y + rows_of(one["residual"])
        outputs.append(back(y, one["x"]))
        if case["train"]:
            density = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi) if act == "gelu" else None
            slope = {"none": lambda: torch.ones_like(z), "relu": lambda: (z > 0).double(),
                     "silu": lambda: logistic * (1 + z - z * logistic), "sigmoid": lambda: logistic - logistic ** 2,
                     "gelu": lambda: normal + z * density}[act]()
            dz = rows_of(one["grad"]) * slope
            outputs += [back(dz @ w, one["x"]), (dz.t() @ x).view(one["weight"].shape), dz.sum(0)]
    return outputs
