"""Label probabilities at bounds that do not grow with the number of classes and that are relative to what they bound
(derived in label_probs_bounds.py)."""
import math

import pytest
import torch

from label_probs_bounds import Row, within
from ldmseg.ops import native as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _row(kind, C, gen):
    if kind == "equal":
        return torch.zeros(C)
    if kind == "gap":                       # one class against all others, together as likely as it
        x = torch.full((C,), -math.log(C))
        x[C // 3] = 0.0
        return x
    if kind == "far_gap":
        x = torch.full((C,), -15.0)
        x[-1] = 0.0
        return x
    if kind == "rising":
        return torch.arange(C) * 1e-6
    if kind == "rising_fast":
        return torch.arange(C) * 1e-4
    if kind == "falling":
        return torch.arange(C) * -1e-5
    return torch.randn(C, generator=gen) * 2


KINDS = ["equal", "gap", "far_gap", "rising", "rising_fast", "falling", "normal"]


def _check_forward(x, y, dim, topk, mask=None, temperature=1.0):
    out = K.label_log_probs(x, y, dim=dim, topk=topk, class_mask=mask, temperature=temperature, want_stats=True)
    row = Row(x, dim, temperature, mask)
    within(out.entropy, row.H, row.err_H(), "entropy")
    ids = y.unsqueeze(-1)
    within(out.log_prob.unsqueeze(-1), row.log_p(ids), row.err_log_p(ids), "log_prob")
    if topk:
        ids = out.top_ids.movedim(dim, -1).long()
        within(out.top_log_probs.movedim(dim, -1), row.log_p(ids), row.err_log_p(ids), "top_log_probs")
    return out, row


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("C", [700, 4096, 16384, 50001, 131072])
def test_sums_over_many_strided_classes(C, dtype):
    """Equal gaps round in one direction all the way, and a rising row moves its maximum at every class: neither may
    show in the sums as their number grows."""
    g = torch.Generator().manual_seed(C)
    N = 70 if C <= 4096 else 10                                 # enough of them for a list of the classes left
    x = torch.stack([_row(k, C, g) for k in KINDS]).to(DT[dtype]).unsqueeze(2).expand(-1, -1, N).contiguous().to(DEV)
    y = torch.randint(0, C, (len(KINDS), N), generator=g).to(DEV)
    _check_forward(x, y, 1, 3)
    mask = torch.rand(len(KINDS), C, generator=g) < 0.8
    mask[:, C // 3] = True
    mask.scatter_(1, y.cpu(), True)
    _check_forward(x, y, 1, 0, mask.to(DEV))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("masked", [False, True])
def test_sums_with_a_thread_to_a_position(masked, dtype):
    """131200 positions of 2048 classes: one thread has all classes of a position.  Every position has the same row."""
    C, N = 2048, 131200
    g = torch.Generator().manual_seed(1)
    for kind in ("equal", "gap", "rising"):
        one = _row(kind, C, g).to(DT[dtype]).to(DEV)
        mask = None
        if masked:
            mask = torch.ones(1, C, dtype=torch.bool, device=DEV)
            mask[:, 5::3] = False
            mask[:, C // 3] = True
        out = K.label_log_probs(one.view(1, C, 1).expand(1, C, N).contiguous(),
                                torch.full((1, N), C // 3, device=DEV), class_mask=mask)
        row = Row(one.view(1, C, 1), 1, class_mask=mask)
        ids = torch.full((1, 1, 1), C // 3, device=DEV)
        for at in (0, 1, N // 2, N - 1):
            within(out.entropy[:, at:at + 1], row.H, row.err_H(), "entropy")
            within(out.log_prob[:, at:at + 1, None], row.log_p(ids), row.err_log_p(ids), "log_prob")
        assert (out.entropy == out.entropy[0, 0]).all() and (out.log_prob == out.log_prob[0, 0]).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("C,N", [(1001, 7), (8192, 2051), (20000, 600), (1_000_003, 7)])
def test_sums_over_many_adjacent_classes(C, N, dtype):
    g = torch.Generator().manual_seed(C)
    x = torch.stack([_row(k, C, g) for k in KINDS]).to(DT[dtype]).to(DEV)
    x = x.repeat(-(-N // len(KINDS)), 1)[:N]
    y = torch.randint(0, C, (N,), generator=g).to(DEV)
    if N * C > 1 << 24:                                         # only some of the rows' references fit
        out = K.label_log_probs(x, y)
        keep = torch.cat([torch.arange(7), torch.arange(N - 7, N)]).to(DEV)
        row, ids = Row(x[keep]), y[keep, None]
        within(out.entropy[keep], row.H, row.err_H(), "entropy")
        within(out.log_prob[keep, None], row.log_p(ids), row.err_log_p(ids), "log_prob")
    else:
        _check_forward(x, y, 1, 3)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("layout", ["planes", "planes_odd", "short_rows", "rows", "long_rows"])
@pytest.mark.parametrize("T", [1.0, 0.5])
def test_gradient_of_a_confident_label_keeps_its_digits(layout, T, dtype):
    """1 - p of the label runs from 0.3 to 1e-12: its gradient is relative to that, also below a rounding of 1, and
    the row's gradients add up to 0 as far as their type can say."""
    C = {"planes": 37, "planes_odd": 37, "short_rows": 40, "rows": 700, "long_rows": 3001}[layout]
    N = 62 if layout != "planes_odd" else 61
    g = torch.Generator().manual_seed(C)
    gaps = torch.linspace(2.0, 30.0, N) + math.log(C)
    x = -gaps.unsqueeze(1) - 2 * torch.rand(N, C, generator=g)
    y = torch.randint(0, C, (N,), generator=g)
    x.scatter_(1, y.unsqueeze(1), 0.0)
    x = (x * T).to(DT[dtype])
    y[-1] = (y[-1] + 1) % C                                     # one that is not the maximum
    x[5, (y[5] + 1) % C] = 0.0                                  # two maxima
    gl = torch.randn(N, generator=g)
    ge = torch.randn(N, generator=g)
    ge[::2] = 0
    if layout.startswith("planes"):
        xx, yy, dim = x.t().contiguous().unsqueeze(0).to(DEV), y.unsqueeze(0).to(DEV), 1
        gl, ge = gl.unsqueeze(0), ge.unsqueeze(0)
    else:
        xx, yy, dim = x.to(DEV), y.to(DEV), 1
    gl, ge = gl.to(DEV), ge.to(DEV)
    out = K.label_log_probs(xx, yy, temperature=T, want_stats=True)
    for e in (None, ge):
        d = K.label_log_probs_bwd(xx, out.stats, gl, e, temperature=T)
        want, tol = Row(xx, dim, T).grad(yy, gl.double(), None if e is None else e.double(), xx.dtype)
        got = d.movedim(dim, -1)
        own = torch.zeros_like(want, dtype=torch.bool).scatter_(-1, yy.unsqueeze(-1), True)
        within(got[own], want[own], tol[own], "the label's gradient")
        within(got, want, tol, "gradient")
        if e is None:
            assert ((got.double().sum(-1)).abs() <= tol.sum(-1)).all()
            assert (got[own] != 0).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("C,N,masked", [(600_000, 32, False), (600_000, 3, True), (1 << 21, 2, False), (530_000, 70, True)])
def test_gradient_of_many_strided_classes(C, N, masked, dtype):
    """More classes than 65535 spans of 8, for fewer positions than a wave: the backward takes what the forward does."""
    g = torch.Generator(device=DEV).manual_seed(C)
    x = (torch.randn(1, C, N, device=DEV, generator=g) * 3)
    x[0, C - 1, 0] = x[0, 5, 0] = 30.0
    x = x.to(DT[dtype])
    y = torch.randint(0, C, (1, N), device=DEV, generator=g)
    y[0, 0] = C - 1
    mask = None
    if masked:
        mask = torch.rand(1, C, device=DEV, generator=g) < 0.7
        mask[0, y[0]] = True
    gl, ge = (torch.randn(1, N, device=DEV, generator=g) for _ in range(2))
    out, row = _check_forward(x, y, 1, 2, mask)
    d = K.label_log_probs_bwd(x, out.stats, gl, ge, class_mask=mask)
    want, tol = row.grad(y, gl.double(), ge.double(), x.dtype)
    within(d.movedim(1, -1), want, tol, "gradient")
    assert mask is None or (d[0, ~mask[0]] == 0).all()


def test_lazily_negated_tensors_are_read_as_they_are():
    """The imaginary part of a conjugate is a view that torch negates as it reads: logits and arriving gradients of that
    kind have their own sign."""
    g = torch.Generator().manual_seed(7)

    def view(*shape):
        v = torch.complex(torch.randn(*shape, generator=g), torch.randn(*shape, generator=g)).to(DEV).conj().imag
        assert v.is_neg()
        return v

    for shape in ((2, 19, 33), (40, 300), (1, 7, 1)):
        x, y = view(*shape), torch.randint(0, shape[1], shape[:1] + shape[2:], generator=g).to(DEV)
        gl, ge = view(*y.shape), view(*y.shape)
        out, ref = (K.label_log_probs(v, y, topk=3, want_stats=True) for v in (x, x.resolve_neg().contiguous()))
        assert torch.equal(out.top_ids, ref.top_ids)
        assert (out.log_prob - ref.log_prob).abs().max() < 1e-5 and (out.entropy - ref.entropy).abs().max() < 1e-5
        d = K.label_log_probs_bwd(x, out.stats, gl, ge)
        want = K.label_log_probs_bwd(x.resolve_neg().contiguous(), ref.stats, gl.resolve_neg(), ge.resolve_neg())
        assert (d - want).abs().max() < 1e-5
    one = torch._neg_view(torch.randn(1, 5, 1, generator=g).to(DEV))
    assert torch.equal(K.label_log_probs(one).entropy, K.label_log_probs(one.resolve_neg()).entropy)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape,T,masked", [
    ((5, 7), 1.0, False), ((513, 30), 1.0, True), ((3, 1023), 0.7, False), ((4, 1025), 1.0, False), ((70, 5000), 1.0, True),
    ((70, 5000), 1.0, False), ((1, 16385), 1.0, False), ((3, 40001), 0.7, True), ((1, 131072), 1.0, False),
    ((2051, 2001), 1.0, False), ((9, 2041), 1.0, False), ((300, 4099), 2.0, True),
    ((2, 30, 24, 80), 1.0, False), ((1, 128, 37, 53), 1.0, True), ((2, 33, 17, 31), 0.7, False), ((1, 513, 3, 67), 1.0, False),
    ((3, 19, 8, 8), 1.0, True), ((2, 70, 64, 66), 0.5, False),
])
def test_gradient_element_by_element(shape, T, masked, dtype):
    """Every element against a bound of its own size: most are far below the largest of their row, and neither they nor a
    row's last ones could be left out or swapped unseen."""
    g = torch.Generator().manual_seed(sum(shape))
    N, C = shape[:2]
    x = (torch.randn(shape, generator=g) * 3).to(DT[dtype]).to(DEV)
    y = torch.randint(0, C, shape[:1] + shape[2:], generator=g)
    y = torch.where(torch.rand(y.shape, generator=g) < 0.3, x.argmax(1).cpu(), y).to(DEV)
    mask = None
    if masked:
        mask = torch.rand(N, C, generator=g) < 0.7
        mask[:, 0] = True
        y = torch.where(mask.to(DEV).view(N, C, *[1] * (x.ndim - 2)).expand(x.shape).gather(1, y.unsqueeze(1))[:, 0], y, 0)
        mask = mask.to(DEV)
    gl, ge = (torch.randn(y.shape, generator=g).to(DEV) for _ in range(2))
    out, row = _check_forward(x, y, 1, 0, mask, T)
    for a, b in ((gl, None), (None, ge), (gl, ge)):
        got = K.label_log_probs_bwd(x, out.stats, a, b, temperature=T, class_mask=mask).movedim(1, -1)
        want, tol = row.grad(y, a if a is None else a.double(), b if b is None else b.double(), x.dtype)
        if masked:
            left = mask.view(N, *[1] * (x.ndim - 2), C).expand(want.shape)
            assert (got[~left] == 0).all()
        else:
            left = torch.ones_like(want, dtype=torch.bool)
        # the bound tells: twice it is less than the element, nearly everywhere and in the last classes too
        tells = (2 * tol < want.abs()) | ~left
        assert tells.double().mean() > 0.9 and tells[..., -16:].double().mean() > 0.9
        within(got, want, tol, "gradient")


def test_rows_past_32_bits_of_elements():
    """2.2e6 rows of 1000 bf16 classes in a matrix of 2.2e9 elements: both ends, forward and backward."""
    if torch.cuda.get_device_properties(0).total_memory < 40e9:
        pytest.skip("needs 20 GB")
    g = torch.Generator().manual_seed(3)
    N, C = 2_200_000, 1000
    x = torch.zeros(N, C + 1, dtype=torch.bfloat16, device=DEV)[:, :C]
    ends = torch.tensor([0, 1, N // 2, N - 3, N - 2, N - 1], device=DEV)
    x[ends[1:]] = torch.randn(5, C, generator=g).bfloat16().to(DEV)
    y = torch.zeros(N, dtype=torch.int64, device=DEV)
    y[ends] = torch.tensor([3, 999, 17, 0, 501, 998], device=DEV)
    out = K.label_log_probs(x, y, topk=2, want_stats=True)
    row, ids = Row(x[ends]), y[ends, None]
    within(out.entropy[ends], row.H, row.err_H(), "entropy")
    within(out.log_prob[ends, None], row.log_p(ids), row.err_log_p(ids), "log_prob")
    assert abs(out.log_prob[0].item() + math.log(C)) < 1e-4 and abs(out.log_prob[5].item() + math.log(C)) < 1e-4
    assert torch.equal(out.top_ids[ends[1:]].long(), x[ends[1:]].float().topk(2, dim=1).indices)
    gl = torch.ones(N, device=DEV)
    gl[ends] = torch.randn(6, generator=g).to(DEV)
    d = K.label_log_probs_bwd(x, out.stats, gl)
    want, tol = row.grad(y[ends], gl[ends].double(), None, x.dtype)
    within(d[ends], want, tol, "gradient")
