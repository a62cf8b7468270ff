"""Gradient clipping for training loops whose gradients are separate tensors: ``loss.backward()`` on the
drop-in UNet or any other module, as in the reference's update_weights (trainers_ldm_cond.py:769-781).
The native training steps keep ONE flat gradient and clip inside their fused AdamW instead."""
import torch

from ..ops import native as K


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ on the HIP path: the global norm of all gradients, then every gradient
    times min(1, max_norm / (norm + 1e-6)) in place.  Returns the norm before clipping (0-d fp32, on the
    gradients' GPU).

    ``parameters``: a tensor or an iterable of them; those without a gradient are skipped.  Gradients are
    dense fp32 or bf16 on one GPU, in any mix; norm_type 2, inf or 1.  A non-finite norm scales by its
    factor as torch does (inf: 0, NaN: NaN) unless ``error_if_nonfinite``, which raises before anything is
    scaled and is the only form that waits for the GPU.  A gradient listed twice is refused."""
    norm_type = float(norm_type)
    if not error_if_nonfinite:
        r = K._grad_norm(parameters, True, norm_type, max_norm, 1)
        return torch.tensor(0.0) if r is None else r
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    r = K._grad_norm(parameters, True, norm_type, max_norm, 0)
    if r is None:
        return torch.tensor(0.0)
    if not torch.isfinite(r[0]):
        raise RuntimeError(f"the gradients' norm of order {norm_type} is not finite, so they cannot be clipped; "
                           "error_if_nonfinite=False scales them all the same")
    K._grad_norm(parameters, True, norm_type, max_norm, 2, r[1])
    return r[0]
