"""Error bounds of the label-probability kernels that do not grow with the number of classes, element by element.

u = 2^-24 is half a step of fp32; m is the row's maximum, z_j = (x_j - m) / T, p_j its probabilities, A1 = sum p |z| and
A2 = sum p z^2, L = log(sum e^z).
A term e^z: x - m, the constant log2(e) / T, their product and exp2 round, (4 |z| + 5) u of it.  A move of the maximum
multiplies by such a term, |z| e^z <= 0.37: 4 u with its rounding.  Adding up: 16 terms to a chunk, 32 chunks with a move
each in fp32, those in fp64; the last move there 7 and the geometric rest of the moves before it 14; a wave's lanes
6 + 6, a block's waves 3 times 7, segments of a row 2 times 7 in a thread and again 12 and 21 over the block:
16 + 32 * 4 + 21 + 12 + 21 + 14 + 12 + 21 = 245 < K = 256.
  L        (K + 4 A1 + 8 L) u: each term weighs p of the sum, log and reciprocal add a few u of L itself
  log p_y  L's, and 4 |z_y| + 2 |log p_y| for x - m, 1 / T, their product and the difference
  H        L + A1: L's; the terms |z| e^z carry (4 |z| + 8) u, so A1 has 4 A2 + 8 A1 + K A1, and its denominator
           (K + 4 A1) A1 more
The gradient g_l (1[y] - p_j) - g_H p_j (log p_j + H), times 1 / T: p_j = exp2(z2 - log2(e) L) is known to L's error
and (4 |z_j| + 4 L + |log p_j| + 4) u relative; log p_j + H to H's and L's and 4 |z_j| + 2 L + 2 H, absolute; the
factors' products round 6 times.  Everything but the label's own g_l is a multiple of p_j.  The label's g_l (1 - p_y) is
relative to 1 - p_y: for a label at the maximum 1 - p_y is formed from L alone, whose relative error is that of
r = sum over the others, (K + 4 mean |z| of the others + 16) u; for any other 1 - p_y >= 1/2 is a difference from 1.
Results below 2^-126 may be flushed, and one rounding to the logits' type follows."""
import torch

U = 2.0 ** -24
K = 256


class Row:
    """The 64-bit quantities of ``logits`` (any device, classes along dim), classes last, on the logits' device."""

    def __init__(self, logits, dim=1, temperature=1.0, class_mask=None):
        x = logits.detach().double().movedim(dim, -1)
        if class_mask is not None:
            m = class_mask if class_mask.ndim == 1 else class_mask.view(len(class_mask), *[1] * (x.ndim - 2), -1)
            x = x.masked_fill(~m.to(x.device), -torch.inf)
        self.top = x.amax(-1, keepdim=True)
        self.z = (x - self.top) / temperature
        self.at_top = x == self.top
        e = self.z.exp()
        first = torch.zeros_like(e).scatter_(-1, x.argmax(-1, keepdim=True), 1.0)
        r = (e * (1 - first)).sum(-1)
        self.L = torch.log1p(r)
        self.p = e / (1 + r).unsqueeze(-1)
        self.absz = torch.where(self.p > 0, self.z.abs(), torch.zeros_like(e))
        self.A1, self.A2 = (self.p * self.absz).sum(-1), (self.p * self.absz ** 2).sum(-1)
        self.H = self.L + self.A1
        self.others = torch.where(r > 0, (e * (1 - first) * self.absz).sum(-1) / r, torch.zeros_like(r))
        self.T = temperature

    def log_p(self, ids):
        """Of classes [..., k]."""
        return self.z.gather(-1, ids) - self.L.unsqueeze(-1)

    def err_L(self):
        return U * (K + 4 * self.A1 + 8 * self.L)

    def err_H(self):
        return self.err_L() + U * (4 * self.A2 + 8 * self.A1 + K * self.A1 + self.A1 * (K + 4 * self.A1))

    def err_log_p(self, ids):
        z = self.absz.gather(-1, ids)
        return self.err_L().unsqueeze(-1) + U * (4 * z + 2 * (z + self.L.unsqueeze(-1)))

    def grad(self, labels, gl, ge, dtype):
        """-> the gradient and its bound, classes last.  ``labels`` < 0: none; gl, ge fp64 or None."""
        p, z, L, H = self.p, self.absz, self.L.unsqueeze(-1), self.H.unsqueeze(-1)
        zero = torch.zeros_like(self.L)
        gl = (zero if gl is None or labels is None else torch.where(labels >= 0, gl, zero)).unsqueeze(-1)
        ge = (zero if ge is None else ge).unsqueeze(-1)
        own = torch.zeros_like(p)
        if labels is not None:
            own.scatter_(-1, labels.clamp(min=0).unsqueeze(-1), 1.0)
            own *= (labels >= 0).unsqueeze(-1)
        # 1 - p without the difference: L is log1p(r), so 1 - 1 / (1 + r) is -expm1(-L) at the maximum
        rest = torch.where(self.at_top, -torch.expm1(-L).expand_as(p), 1 - p)
        centred = torch.where(self.at_top, self.A1.unsqueeze(-1).expand_as(p), H - L - z)       # log p + H
        value = own * gl * rest - (1 - own) * gl * p - ge * p * centred
        err_p = self.err_L().unsqueeze(-1) + U * (4 * z + 4 * L + (z + L) + 4)
        err_c = (self.err_H() + self.err_L()).unsqueeze(-1) + U * (4 * z + 2 * L + 2 * H)
        tol = p * ((gl.abs() + ge.abs() * centred.abs()) * (err_p + 6 * U) + ge.abs() * err_c)
        rel = torch.where(self.at_top, (U * (K + 4 * self.others + 16)).unsqueeze(-1) + 0 * p, err_p + 8 * U)
        tol = torch.where(own > 0, gl.abs() * rest * rel + p * ge.abs() * (centred.abs() * (err_p + 6 * U) + err_c), tol)
        value, tol = value / self.T, tol / self.T
        tol = tol + 2.0 ** -125 * (gl.abs() + ge.abs() * (1 + centred.abs())) / self.T
        half = torch.finfo(dtype).eps / 2
        return value, tol * (1 + half) + half * value.abs() + 2.0 ** -133


def within(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert got.isfinite().all(), what
    worst = ((got - want).abs() / tol).max().item()
    assert worst <= 1, f"{what}: {worst:.3g} times the bound"
