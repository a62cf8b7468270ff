"""``label_log_probs`` as an autograd node: log probabilities of given labels and entropies of every position of
class logits, differentiable in the logits, with the most likely alternatives (ops.native has the launches)."""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import native as K


class _LabelLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, dim, topk, temperature, ignore_label, class_mask):
        out = K.label_log_probs(logits, labels, dim=dim, topk=topk, temperature=temperature,
                                ignore_label=ignore_label, class_mask=class_mask, want_stats=True)
        ctx.save_for_backward(logits, out.stats, class_mask)
        ctx.dim, ctx.temperature = dim, temperature
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*[t for t in (out.top_log_probs, out.top_ids) if t is not None])
        return out.log_prob, out.entropy, out.top_log_probs, out.top_ids

    @staticmethod
    @once_differentiable
    def backward(ctx, d_log_prob, d_entropy, *_):
        logits, stats, class_mask = ctx.saved_tensors
        d = None
        if d_log_prob is not None or d_entropy is not None:
            d = K.label_log_probs_bwd(logits, stats, d_log_prob, d_entropy, dim=ctx.dim, temperature=ctx.temperature,
                                      class_mask=class_mask)
        return d, None, None, None, None, None, None


def label_log_probs(logits, labels=None, *, dim=1, topk=0, temperature=1.0, ignore_label=None, class_mask=None):
    """ops.native.label_log_probs with gradients: ``log_prob`` and ``entropy`` of the result are differentiable
    in ``logits`` (the alternatives are not), backward and once.  Without a gradient to take it saves nothing for one.

        nll = -label_log_probs(logits, labels, ignore_label=255).log_prob.sum() / (labels != 255).sum()
        nll.backward()
    """
    if forward_ad.unpack_dual(logits).tangent is not None:
        raise NotImplementedError("label_log_probs has no forward-mode derivative: take its gradient backward, or call "
                                  "it on logits without a tangent")
    if torch.is_grad_enabled() and logits.requires_grad:
        return K.LabelProbs(*_LabelLogProbs.apply(logits, labels, dim, topk, temperature, ignore_label, class_mask),
                            None)
    return K.label_log_probs(logits, labels, dim=dim, topk=topk, temperature=temperature, ignore_label=ignore_label,
                             class_mask=class_mask)
