"""Plain 64-bit restatement of the label-probability operator: log probability of a given label, entropy and the
most likely classes of softmax(logits / T), and the gradient of the first two.  Loops over nothing, shares nothing
with the kernels."""
import torch

INF = float("inf")


def _left(logits, dim, class_mask):
    """bool like ``logits`` (classes last): the classes that a row may use."""
    x = logits.detach().double().cpu().movedim(dim, -1)
    if class_mask is None:
        return x, torch.ones_like(x, dtype=torch.bool)
    m = class_mask.cpu()
    if m.ndim == 2:
        m = m.view(m.shape[0], *[1] * (x.ndim - 2), m.shape[1])
    return x, m.expand(x.shape)


def label_log_probs(logits, labels=None, *, dim=1, topk=0, temperature=1.0, ignore_label=None, class_mask=None):
    """-> dict of fp64 / int64 CPU tensors: log_prob, entropy, top_log_probs, top_ids (classes' dim where the
    operator has it) and log_p, the whole distribution with the classes last."""
    x, left = _left(logits, dim, class_mask)
    C = x.shape[-1]
    z = torch.where(left, x / temperature, torch.full_like(x, -INF))
    some = (z > -INF).any(-1, keepdim=True) | z.isnan().any(-1, keepdim=True)
    bad = z.isnan().any(-1, keepdim=True) | (z == INF).any(-1, keepdim=True)
    m = torch.where(some & ~bad, z.amax(-1, keepdim=True), torch.zeros_like(z[..., :1]))
    log_p = (z - m) - (z - m).exp().sum(-1, keepdim=True).log()
    log_p = torch.where(some, log_p, torch.full_like(z, -INF))
    log_p = torch.where(bad, torch.full_like(z, float("nan")), log_p)
    p = log_p.exp()
    ent = -torch.where(p == 0, torch.zeros_like(p), p * log_p).sum(-1)
    out = {"log_p": log_p, "entropy": ent}
    if labels is not None:
        y = labels.cpu()
        inside = (y >= 0) & (y < C)
        lp = log_p.gather(-1, y.clamp(0, C - 1).unsqueeze(-1)).squeeze(-1)
        lp = torch.where(inside, lp, torch.full_like(lp, float("nan")))
        if ignore_label is not None:
            lp = torch.where(y == ignore_label, torch.zeros_like(lp), lp)
        out["log_prob"] = lp
    if topk:
        v = torch.where(left, x, torch.full_like(x, -INF))
        rank = torch.where(v.isnan(), torch.full_like(v, INF), v)
        # NaN first, then by value; a stable sort keeps the lower class first
        order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
        nan_first = torch.sort(v.isnan().to(torch.int8).gather(-1, order), dim=-1, descending=True, stable=True).indices
        ids = order.gather(-1, nan_first)[..., :topk]
        gone = v.gather(-1, ids) == -INF
        out["top_ids"] = torch.where(gone, torch.full_like(ids, -1), ids).movedim(-1, dim)
        out["top_log_probs"] = torch.where(gone, torch.full_like(ids, 0).double() - INF,
                                           log_p.gather(-1, ids)).movedim(-1, dim)
    return out


def label_log_probs_bwd(logits, labels, d_log_prob, d_entropy, *, dim=1, temperature=1.0, ignore_label=None,
                        class_mask=None):
    """d logits in fp64, from the formula (not by autograd)."""
    f = label_log_probs(logits, labels, dim=dim, temperature=temperature, ignore_label=ignore_label,
                        class_mask=class_mask)
    log_p, C = f["log_p"], f["log_p"].shape[-1]
    p = log_p.exp()
    d = torch.zeros_like(p)
    if d_log_prob is not None and labels is not None:
        y = labels.cpu()
        ok = (y >= 0) & (y < C) & (f["log_prob"] > -INF)
        if ignore_label is not None:
            ok &= y != ignore_label
        g = torch.where(ok, d_log_prob.double().cpu(), torch.zeros(y.shape, dtype=torch.float64)).unsqueeze(-1)
        one = torch.zeros_like(p).scatter_(-1, y.clamp(0, C - 1).unsqueeze(-1), 1.0)
        d += g * (one - p)
    if d_entropy is not None:
        h = f["entropy"].unsqueeze(-1)
        d -= d_entropy.double().cpu().unsqueeze(-1) * torch.where(p == 0, torch.zeros_like(p), p * (log_p + h))
    left = _left(logits, dim, class_mask)[1]
    return torch.where(left, d / temperature, torch.zeros_like(d)).movedim(-1, dim)
