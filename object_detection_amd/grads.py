"""The norm of all gradients of a training step taken as one vector, and clipping by it.

What stands between ComputeLoss / the layers' gradients and the optimizer in a step of object_detection/yolov5/train.py:337-346
(scaler.scale(loss).backward(); scaler.step(optimizer)): the gradients carry a loss scale there, which both calls can take out on
the way.  Two launches for up to 120 tensors of one type, no host synchronisation, sums in double, results repeat bit for bit.
"""
from array import array

import torch

from . import _lib as L
from .dist import all_reduce_norm_power

_NORMS = {1.0: 1, 2.0: 2, float("inf"): 0}
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
# read per tensor with map(): a list of a hundred gradients costs a few microseconds for each of these
_data_ptr, _numel, _is_contiguous, _device_of, _dtype_of = (torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_contiguous,
                                                            torch.Tensor.get_device, torch.Tensor.dtype.__get__)


def _norm_code(where, norm_type):
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise ValueError(f"{where}: norm_type must be 1, 2 or inf, got {norm_type}")
    return code


def _limit(where, max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"{where}: max_norm must not be negative, got {max_norm}")
    return max_norm


def _dense(t):
    """t as the kernels read it: its elements in one piece, in any order of the axes (a channels_last gradient stays)."""
    if t.layout != torch.strided:
        raise RuntimeError(f"gradients must be dense tensors, got {t.layout}")
    if t.is_contiguous() or (t.dim() == 4 and t.is_contiguous(memory_format=torch.channels_last)):
        return t
    return t.contiguous()


def _checked(where, grads):
    """The list split by type: [(type, indices)], and the one device."""
    try:
        devices, kinds = set(map(_device_of, grads)), set(map(_dtype_of, grads))
    except TypeError:
        raise TypeError(f"{where}: gradients must be tensors, got {[type(g).__name__ for g in grads if not isinstance(g, torch.Tensor)][:3]}") from None
    if -1 in devices:
        raise RuntimeError(f"{where}: a gradient is on the CPU: object_detection_amd only runs on ROCm devices (no CPU fallback)")
    if len(devices) != 1:
        raise RuntimeError(f"{where}: gradients are on several devices: {sorted(devices)}")
    if not kinds <= _DTYPES.keys():
        raise RuntimeError(f"{where}: gradients must be fp32, fp16 or bf16, got {kinds - _DTYPES.keys()}")
    if len(kinds) == 1:
        return [(kinds.pop(), None)], grads[0].device
    return [(k, [i for i, g in enumerate(grads) if g.dtype == k]) for k in sorted(kinds, key=_DTYPES.get)], grads[0].device


def _scale_on(scale, device, where):
    """The loss scale as one device float, or None."""
    if scale is None:
        return None
    if isinstance(scale, torch.Tensor):
        if scale.numel() != 1:
            raise RuntimeError(f"{where}: scale must be one number, got shape {tuple(scale.shape)}")
        return scale.detach().to(device=device, dtype=torch.float32)
    return None if scale == 1 else torch.full((), float(scale), dtype=torch.float32, device=device)


class _List:
    """One type's tensors as the C entries take them."""
    __slots__ = ("dtype", "pointers", "sizes", "count", "parts", "keep")

    def __init__(self, dtype, tensors):
        self.dtype, self.keep = dtype, tensors
        self.pointers = array("Q", map(_data_ptr, tensors))
        self.sizes = array("q", map(_numel, tensors))
        self.count = len(tensors)
        self.parts = L.lib().dh_grad_parts(_at(self.sizes), self.count)


def _at(a):
    return a.buffer_info()[0]


def _powers(lists, code, device):
    """The partial sums of every list, one after the other."""
    partial = torch.empty(sum(t.parts for t in lists), dtype=torch.float64, device=device)
    lib, at, st = L.lib(), partial.data_ptr(), L.raw_stream()
    for t in lists:
        L.check(lib.dh_grad_power(_at(t.pointers), _at(t.sizes), t.count, _DTYPES[t.dtype], code, at, t.parts, st), "dh_grad_power")
        at += 8 * t.parts
    return partial


def _over_group(partial, code, norm_type, group):
    """The ranks' powers joined: one part instead of this rank's."""
    power = torch.empty(1, dtype=torch.float64, device=partial.device)
    L.check(L.lib().dh_grad_norm(partial.data_ptr(), partial.numel(), code, None, power.data_ptr(), None, L.raw_stream()), "dh_grad_norm")
    return all_reduce_norm_power(power, float(norm_type), None if group is True else group)


def total_grad_norm(grads, norm_type=2.0, scale=None, group=None):
    """The norm of all `grads` as one vector: a 0-dim fp32 tensor on their device (0 on the CPU for an empty list).

    norm_type 1, 2 or inf; scale: a factor the gradients carry (GradScaler's, a number or a one-element tensor) and the norm is
    to be free of.  group: a process group (True: the default one) over which gradients are sharded -- every rank passes its own
    shards and gets the norm of all of them; leave it out for replicated gradients."""
    code, grads = _norm_code("total_grad_norm", norm_type), list(grads)
    if not grads and group is None:
        return torch.zeros(())
    if not grads:
        raise RuntimeError("total_grad_norm: a rank of a group needs at least one gradient (it may be empty)")
    by_type, device = _checked("total_grad_norm", grads)
    norm = torch.empty((), dtype=torch.float32, device=device)
    with torch.no_grad(), L.device_guard(device):
        factor = _scale_on(scale, device, "total_grad_norm")
        lists = [_List(t, [_dense(g) for g in (grads if at is None else [grads[i] for i in at])]) for t, at in by_type]
        partial = _powers(lists, code, device)
        if group is not None:
            partial = _over_group(partial, code, norm_type, group)
        L.check(L.lib().dh_grad_norm(partial.data_ptr(), partial.numel(), code, L.ptr(factor), None, norm.data_ptr(), L.raw_stream()), "dh_grad_norm")
    return norm


def _no_overlap(where, some, pointers):
    """A tensor that two workgroups would scale at once: the same output twice, or an output that is another gradient."""
    outs = set(pointers)
    if len(outs) != some.count and len({p for p, n in zip(pointers, some.sizes) if n}) != sum(n > 0 for n in some.sizes):
        raise RuntimeError(f"{where}: a gradient is in the list twice")
    if pointers is not some.pointers and not outs.isdisjoint(some.pointers):
        own = {p: k for k, p in enumerate(some.pointers) if some.sizes[k]}
        if any(own.get(p, k) != k for k, p in enumerate(pointers) if some.sizes[k]):
            raise RuntimeError(f"{where}: an output is another gradient of the list")


def _contiguous(tensors):
    try:
        return all(map(_is_contiguous, tensors))
    except RuntimeError:                     # a layout that has no such notion
        return False


def _clip(where, grads, outs, max_norm, norm_type, scale, group):
    """Norm, and outs[k] = grads[k] / scale * factor; outs[k] may be grads[k]."""
    code, max_norm = _norm_code(where, norm_type), _limit(where, max_norm)
    by_type, device = _checked(where, grads)
    in_place = outs is grads
    plain = _contiguous(grads) and (in_place or _contiguous(outs))
    with torch.no_grad(), L.device_guard(device):
        factor = _scale_on(scale, device, where)
        norm = torch.empty((), dtype=torch.float32, device=device)
        # tensors whose elements are not in one piece, or not in the same order in both: through copies
        sources = grads if plain else [_dense(g) for g in grads]
        if plain:
            targets = outs
        else:
            targets = [o if o.shape == s.shape and o.stride() == s.stride() and _dense(o) is o else torch.empty_like(s, dtype=o.dtype) for s, o in zip(sources, outs)]
        lists = [_List(t, sources if at is None else [sources[i] for i in at]) for t, at in by_type]
        into = []                            # per list: [(output type, list, pointers)]
        for t, (dtype, at) in zip(lists, by_type):
            mine = targets if at is None else [targets[i] for i in at]
            kinds = {dtype} if in_place and plain else set(map(_dtype_of, mine))
            if len(kinds) == 1:
                groups = [(kinds.pop(), t, t.pointers if in_place and plain else array("Q", map(_data_ptr, mine)))]
            else:                            # both kinds of outputs for one kind of gradients
                groups = []
                for d in (dtype, torch.float32):
                    pick = [k for k, o in enumerate(mine) if o.dtype == d]
                    groups.append((d, _List(dtype, [t.keep[k] for k in pick]), array("Q", [mine[k].data_ptr() for k in pick])))
            for d, some, pointers in groups:
                _no_overlap(where, some, pointers)
            into.append(groups)
        partial = _powers(lists, code, device)
        if group is not None:
            partial = _over_group(partial, code, norm_type, group)
        lib, st = L.lib(), L.raw_stream()
        for t, groups in zip(lists, into):
            for d, some, pointers in groups:
                L.check(lib.dh_grad_clip(_at(some.pointers), _at(pointers), _at(some.sizes), some.count, _DTYPES[t.dtype], _DTYPES[d], code,
                                         partial.data_ptr(), partial.numel(), L.ptr(factor), max_norm, norm.data_ptr(), st), "dh_grad_clip")
        if not plain:
            for o, t in zip(outs, targets):
                if t is not o:
                    o.copy_(t if t.shape == o.shape else t.reshape(o.shape))
    torch.autograd.graph.increment_version(outs)       # written through raw pointers: keep the version counters honest
    return norm


def clip_grads(grads, max_norm, norm_type=2.0, scale=None, out=None, group=None):
    """(norm, out): the norm of all gradients and the gradients scaled to it, out[k] = grads[k] / scale * min(1, max_norm /
    (norm + 1e-6)).

    grads stay as they are; out is a list of tensors with as many elements, of the gradients' type or fp32 (a master buffer's views),
    made like the gradients if not given; an entry may be the gradient itself.  norm_type, scale and group as in
    total_grad_norm().  A norm that is not finite (an overflowed step under a loss scale) shows in `norm`; the outputs are then
    worthless, as after torch's clipping."""
    grads = list(grads)
    if not grads:
        raise RuntimeError("clip_grads: no gradients")
    _norm_code("clip_grads", norm_type), _limit("clip_grads", max_norm)
    if out is None:
        _checked("clip_grads", grads)
        out = [torch.empty_like(g) for g in grads]
    else:
        out = list(out)
        if len(out) != len(grads):
            raise RuntimeError(f"clip_grads: {len(grads)} gradients and {len(out)} outputs")
        try:
            same = list(map(_numel, grads)) == list(map(_numel, out)) and set(map(_device_of, out)) == {grads[0].get_device()}
            kinds = set(map(_dtype_of, out))
        except (AttributeError, TypeError):
            raise TypeError("clip_grads: gradients and outputs must be tensors") from None
        if same and kinds != {torch.float32}:
            same = all(o.dtype in (g.dtype, torch.float32) for g, o in zip(grads, out))
        if not same:
            raise RuntimeError("clip_grads: an output must have its gradient's number of elements and device, and its type or fp32")
    return _clip("clip_grads", grads, out, max_norm, norm_type, scale, group), out


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, scale=None, group=None):
    """torch.nn.utils.clip_grad_norm_ on the .grad of the given parameters, in place -> the norm before clipping.

    parameters: an iterable of tensors or one tensor; those without a gradient are left out.  Gradients whose norm is below
    max_norm are not written.  error_if_nonfinite reads the norm on the host and raises before anything is scaled; otherwise there is
    no synchronisation.  scale, group: as in total_grad_norm() (with a scale the gradients come out unscaled)."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = [g for g in [p.grad for p in parameters] if g is not None]
    if not grads:
        return torch.zeros(())
    if error_if_nonfinite:
        norm = total_grad_norm(grads, norm_type, scale, group)
        if not torch.isfinite(norm):
            raise RuntimeError(f"clip_grad_norm_: the norm of order {norm_type} of the gradients is {float(norm)}: not finite")
    return _clip("clip_grad_norm_", grads, grads, max_norm, norm_type, scale, group)
