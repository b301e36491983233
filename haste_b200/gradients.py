"""The norm of all gradients of a training step, and clipping by it.

    norm = gradients.clip_grad_norm_(net.parameters(), 1.0)      # scales p.grad in place
    norm = gradients.clip_gradients(grads, 1.0, out=masters)     # scales into other tensors, of other types
    norm = gradients.grad_norm(grads)

norm = sqrt(sum of squares over all tensors), a float32 scalar on their device.  Up to 64 squares at a time are added in float32,
again in 64 bits where their sum leaves 1e-20 to 1e30, so that neither large nor small gradients leave float32's range on the
way; those sums are added in 64 bits, in a fixed order.  The norm is within 10.5 roundings of float32 (2^-24 each).  Gradients
are multiplied by min(1, max_norm / (norm + 1e-6)).  Tensors are float32, bfloat16 or float16, in any mixture, on one GPU, and
fill one range of memory each, in any order of axes.  The calls run on the current stream, never wait for the device (unless
`error_if_nonfinite` asks for it), and may be captured in graphs.  The reference has no counterpart of them.
"""
import torch

from . import _C

__all__ = ["grad_norm", "clip_gradients", "clip_grad_norm_"]


_native = _C.native


def _tensors(gradients):
    return [gradients] if torch.is_tensor(gradients) else [g for g in gradients if g is not None]


def grad_norm(gradients):
    """The norm of a tensor or of several (those that are None count as zero)."""
    some = _tensors(gradients)
    return _native().clip_gradients(some, None, None) if some else torch.zeros(())


def clip_gradients(gradients, max_norm, out=None):
    """Scales the gradients so that their norm is at most `max_norm` (a factor of 1 where that is infinite), in place or,
    where given, into `out`: tensors of the same shapes that lie in memory alike, of any of the three types.  No two may
    overlap in memory; in place, a tensor that is listed twice counts once.  Returns the norm before.

    A norm that is not finite scales as the formula says: an infinite one to zero (infinite values to NaN), NaN to NaN."""
    if out is not None:
        gradients, out = ([t] if torch.is_tensor(t) else list(t) for t in (gradients, out))
        return _native().clip_gradients(gradients, max_norm, out) if gradients or out else torch.zeros(())
    some = _tensors(gradients)
    return _native().clip_gradients(some, max_norm, None) if some else torch.zeros(())


def clip_grad_norm_(parameters, max_norm, error_if_nonfinite=False):
    """`clip_gradients` over the `.grad` of a parameter or of several; a parameter that is listed twice counts once.
    With `error_if_nonfinite` a norm that is not finite raises and leaves the gradients as they are."""
    if torch.is_tensor(parameters):
        parameters = [parameters]
    grads = [p.grad for p in parameters]
    grads = [g for g in grads if g is not None]
    if error_if_nonfinite and grads:
        norm = grad_norm(list({id(g): g for g in grads}.values()))
        if not torch.isfinite(norm):
            raise RuntimeError(f"haste_b200: the norm of the gradients is {norm.item()}; they are not clipped")
    return _native().clip_gradients(grads, max_norm, None) if grads else torch.zeros(())
