"""Shared by the label-probability tests: inputs and the tolerances of the fp32 kernels.

u = 2^-24 is half a step of fp32.  A term e^z, z = (x - m) / T, is one exp2 of a product: x - m, 1 / T, the product
and exp2 round, so its relative error is at most (4 |z| + 2) u; |z| e^z <= 0.37 makes that at most 4 u of the largest
term.  A sum of n of them in sequence adds n u, joining partial sums and following the maximum a few more: the sum
1 + r is known to (n + 32) u, so its log is to (n + 32) u absolute, and log_prob = z_y - log(1 + r) to
(n + 32 + 4 |z_y| + 2 |log_prob|) u.  The entropy's second term carries |z| e^z <= 0.37 per term relative to 1 + r:
the same (n + 32) u times (1 + H).  A gradient g_l (1[y] - p) - g_H p (log p + H) has |p| <= 1 known to
(n + 40 + 4 |log p|) u, p |log p| <= 0.37, and p (log p + H) at most 1 + H: (n + 64) u (|g_l| + |g_H| (1 + H)) / T, and
then one rounding to the logits' type."""
import torch

U = 2.0 ** -24


def chain(logits, dim):
    """Terms that are summed in sequence, at most: every class where they are strided (a thread has a position); of
    adjacent classes 1/256 of them, a row being a block's, and no more than 512 where it is shorter (a wave's 64 lanes
    share up to 8192)."""
    C = logits.shape[dim]
    return C if logits.stride(dim) != 1 or C < 512 else max(512, C // 256 + 64)


def close(got, want, tol, what):
    got = got.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), what + ": NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]) and torch.equal(torch.isinf(got), inf), what + ": infinities"
    ok = torch.isfinite(want)
    off = (got - want).abs()[ok] - (tol.expand(want.shape)[ok] if isinstance(tol, torch.Tensor) else tol)
    assert not off.numel() or off.max() <= 0, f"{what}: {off.max():.3g} over the tolerance"


def check_forward(out, ref, logits, dim, temperature, labels=None, topk=0):
    n = chain(logits, dim)
    H = ref["entropy"]
    close(out.entropy, H, torch.nan_to_num((n + 32) * U * (1 + H)), "entropy")
    if labels is not None:
        lp = ref["log_prob"]
        a = torch.nan_to_num(lp.abs(), nan=0.0, posinf=0.0)
        close(out.log_prob, lp, (n + 32) * U + 6 * U * a + 4 * U * H.nan_to_num(), "log_prob")
    if topk:
        assert torch.equal(out.top_ids.long().cpu(), ref["top_ids"]), "top_ids"
        a = torch.nan_to_num(ref["top_log_probs"].abs(), nan=0.0, posinf=0.0, neginf=0.0)
        close(out.top_log_probs, ref["top_log_probs"], (n + 32) * U + 6 * U * a + 4 * U * H.nan_to_num().amax(),
              "top_log_probs")


def check_grad(got, want, ref, gl, ge, logits, dim, temperature):
    n = chain(logits, dim)
    H = ref["entropy"].nan_to_num()
    g = torch.zeros_like(H)
    if gl is not None:
        g = g + gl.double().cpu().abs()
    if ge is not None:
        g = g + ge.double().cpu().abs() * (1 + H)
    tol = ((n + 64) * U * g / temperature).unsqueeze(dim)
    half = torch.finfo(logits.dtype).eps / 2
    close(got, want, tol + half * want.abs().nan_to_num() * (1 + 1e-6) + 1e-38, "d_logits")
