"""The norm of all gradients of a training step taken as one vector, and clipping by it.

What stands between ComputeLoss / the layers' gradients and the optimizer in a step of object_detection/yolov5/train.py:337-346:
scaler.scale(loss).backward(); scaler.unscale_(optimizer); clip_grad_norm_(...); scaler.step(optimizer).  A GradScaler takes its scale
out itself (in step(), if unscale_() has not), so `scale` stays away from it; `scale` is for loops that multiply the loss, divide by the
scale and skip overflowed steps on their own.  Two launches for up to 280 tensors of one type (176 with other tensors for the results), no host synchronisation, sums
in double, results repeat bit for bit.
"""
import torch

from . import _lib as L
from .dist import all_reduce_norm_power

_NORMS = {1.0: 1, 2.0: 2, float("inf"): 0}


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


def _over(group, norm_type):
    """What joins the ranks' powers, or None."""
    if group is None:
        return None
    return lambda power: all_reduce_norm_power(power, float(norm_type), None if group is True else group)


def _nothing(parameters=()):
    """The empty gradient with which a rank that has none takes part in the exchange the others wait in."""
    return torch.empty(0, device=next((p.device for p in parameters if p.is_cuda), torch.device("cuda")))


def total_grad_norm(grads, norm_type=2.0, scale=None, group=None):
    """The norm of all `grads` as one vector: a 0-dim fp32 tensor on their device (0 on the CPU for an empty list).

    norm_type 1, 2 or inf; scale: a factor the gradients carry (GradScaler's, a number or a one-element tensor) and the norm is
    to be free of.  group: a process group (True: the default one) over which gradients are sharded -- every rank passes its own
    shards (a rank may have none) and gets the norm of all of them; leave it out for replicated gradients."""
    code, grads = _norm_code("total_grad_norm", norm_type), list(grads)
    if not grads and group is None:
        return torch.zeros(())
    return L.host().total_norm(grads or [_nothing()], code, scale, _over(group, norm_type))


def clip_grads(grads, max_norm, norm_type=2.0, scale=None, out=None, group=None):
    """(norm, out): the norm of all gradients and the gradients scaled to it, out[k] = grads[k] / scale * min(1, max_norm /
    (norm + 1e-6)).

    grads stay as they are; out is a list of tensors with as many elements, of the gradients' type or fp32 (a master buffer's views),
    made like the gradients if not given; an entry may be the gradient itself.  norm_type, scale and group as in
    total_grad_norm().  A norm that is not finite (an overflowed step under a loss scale) shows in `norm`; the outputs are then
    worthless, as after torch's clipping."""
    code, limit, grads = _norm_code("clip_grads", norm_type), _limit("clip_grads", max_norm), list(grads)
    if not grads:
        if group is None or out:
            raise RuntimeError("clip_grads: no gradients")
        return total_grad_norm(grads, norm_type, scale, group), []
    if out is None:
        out = [torch.empty_like(g) for g in grads]
    else:
        out = list(out)
    return L.host().clip("clip_grads", grads, out, limit, code, scale, _over(group, norm_type)), out


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, scale=None, group=None):
    """torch.nn.utils.clip_grad_norm_ on the .grad of the given parameters, in place -> the norm before clipping.

    parameters: an iterable of tensors or one tensor; those without a gradient are left out.  Gradients whose norm is below
    max_norm are not written.  error_if_nonfinite reads the norm on the host and raises before anything is scaled; otherwise there is
    no synchronisation.  scale, group: as in total_grad_norm() (with a scale the gradients come out unscaled)."""
    code, limit = _norm_code("clip_grad_norm_", norm_type), _limit("clip_grad_norm_", max_norm)
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    parameters = list(parameters)
    if group is None and not error_if_nonfinite:
        norm = L.host().clip_parameters("clip_grad_norm_", parameters, limit, code, scale, None)
        return torch.zeros(()) if norm is None else norm
    grads = [g for g in [p.grad for p in parameters] if g is not None]
    if not grads and group is not None:         # this rank has nothing to add, the others wait for it all the same
        if not parameters:
            raise RuntimeError("clip_grad_norm_: a rank of a group needs at least one parameter")
        grads = [_nothing(parameters)]
    if not grads:
        return torch.zeros(())
    if error_if_nonfinite:
        norm = total_grad_norm(grads, norm_type, scale, group)
        if not torch.isfinite(norm):
            raise RuntimeError(f"clip_grad_norm_: the norm of order {norm_type} of the gradients is {float(norm)}: not finite")
    return L.host().clip("clip_grad_norm_", grads, None, limit, code, scale, _over(group, norm_type))
