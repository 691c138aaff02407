"""Gradient clipping by the global norm on the device (csrc/grad_clip.hip), the trainer's step between
backward and optimizer (training/trainer.py:118-120).  Nothing waits for the device, except with
error_if_nonfinite."""
from __future__ import annotations

import torch

from .. import _hip


def clip_grads(grads, max_norm, norm_type=2.0, *, inv_scale=None, out=None, error_if_nonfinite=False):
    """Scale the tensors `grads` together so that their global norm is at most max_norm -> the norm before
    clipping, a float32 tensor [].

    The coefficient is min(1, max_norm / (norm + 1e-6)), as torch.nn.utils.clip_grad_norm_ has it, and a
    norm that is not finite acts as it does there (error_if_nonfinite raises before anything is written).
    norm_type: 1, 2 or inf.  inv_scale (one float32 on the device): the reciprocal of a loss scale; the
    gradients are taken times it, in the same pass.  out: tensors to write instead of the gradients, each
    of its gradient's shape and strides and of its type or float32.  The tensors are dense, on one device,
    float32, bfloat16 or float16 in any mixture, and no two of them overlap."""
    grads = list(grads)
    if not grads:
        return torch.tensor(0.0)
    with torch.no_grad():
        if error_if_nonfinite:
            norm = _hip.grad_clip(grads, max_norm, norm_type, inv_scale, out, scale=False)
            if not bool(torch.isfinite(norm)):
                raise RuntimeError(f"the norm of the gradients is {float(norm)}: not clipped")
        return _hip.grad_clip(grads, max_norm, norm_type, inv_scale, out)


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """clip_grads on the .grad of `parameters` (a tensor or an iterable; those without one are left out),
    in place: the arguments and the result of torch.nn.utils.clip_grad_norm_."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    return clip_grads(grads, max_norm, norm_type, error_if_nonfinite=error_if_nonfinite)
