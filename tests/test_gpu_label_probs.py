"""Label probabilities on the HIP path (ldm_label_log_probs, ldm_label_log_probs_bwd) against the 64-bit restatement
in oracle/label_probs.py: layouts, strides, odd sizes, types, masks, degenerate rows, and the gradient."""
import math

import pytest
import torch

from label_probs_utils import check_forward, check_grad
from ldmseg import ops
from ldmseg.ops import native as K
from oracle import label_probs as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
IGN = 255
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _labels(shape, C, gen, logits=None, dim=1):
    y = torch.randint(0, C, shape, generator=gen)
    u = torch.rand(shape, generator=gen)
    if logits is not None:
        y = torch.where(u < 0.5, logits.argmax(dim), y)
    return y.masked_fill(u > 0.9, IGN)


def _run(logits, labels, dim=1, topk=0, temperature=1.0, class_mask=None, gl=True, ge=True, seed=0):
    """Forward and backward of ``logits`` (a GPU tensor, any strides) against the oracle."""
    g = torch.Generator().manual_seed(seed + 99)
    kw = dict(dim=dim, temperature=temperature, class_mask=class_mask)
    out = K.label_log_probs(logits, labels, topk=topk, ignore_label=IGN, want_stats=True, **kw)
    ref = oracle.label_log_probs(logits, labels, topk=topk, ignore_label=IGN, **kw)
    check_forward(out, ref, logits, dim, temperature, labels, topk)
    shape = out.entropy.shape
    dl = torch.randn(shape, generator=g) if gl and labels is not None else None
    de = torch.randn(shape, generator=g) if ge else None
    d = K.label_log_probs_bwd(logits, out.stats, None if dl is None else dl.to(DEV), None if de is None else de.to(DEV),
                              **kw)
    want = oracle.label_log_probs_bwd(logits, labels, dl, de, ignore_label=IGN, **kw)
    assert d.dtype == logits.dtype
    check_grad(d, want, ref, dl, de, logits, dim, temperature)
    return out, d


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("B,C,H,W,topk,T", [
    (1, 1, 1, 1, 1, 1.0),
    (2, 2, 3, 5, 2, 1.0),
    (1, 3, 1, 1, 3, 0.5),
    (2, 7, 1, 63, 4, 2.0),
    (3, 19, 8, 8, 1, 1.0),
    (2, 30, 24, 80, 3, 1.0),
    (1, 30, 1, 257, 0, 0.5),
    (2, 33, 17, 31, 8, 0.7),
    (1, 128, 37, 53, 4, 1.0),
    (4, 128, 64, 64, 5, 1.0),
    (1, 129, 7, 9, 16, 1.0),
    (1, 513, 3, 67, 8, 1.0),
    (1, 31, 200, 211, 2, 1.0),
])
def test_planes(B, C, H, W, topk, T, dtype):
    g = torch.Generator().manual_seed(B * 1000 + C)
    x = (torch.randn(B, C, H, W, generator=g) * 4).to(DT[dtype])
    y = _labels((B, H, W), C, g, x)
    _run(x.to(DEV), y.to(DEV), topk=topk, temperature=T)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("N,C,topk,T", [
    (1, 1, 1, 1.0), (1, 2, 2, 1.0), (3, 3, 2, 1.0), (5, 7, 7, 1.0), (65, 8, 3, 1.0), (7, 9, 4, 0.5), (130, 19, 3, 1.0),
    (513, 30, 3, 1.0), (33, 31, 16, 1.0), (9, 64, 8, 1.0), (1000, 128, 4, 1.0), (5, 255, 5, 2.0), (6, 257, 1, 1.0),
    (3, 1000, 16, 1.0), (3, 1023, 2, 1.0), (4, 1025, 8, 1.0), (2, 2049, 3, 1.0), (1, 4096, 16, 1.0), (70, 5000, 8, 1.0),
    (1, 16385, 8, 1.0), (3, 40001, 4, 0.7), (1, 131072, 16, 1.0), (600, 2500, 1, 1.0),
])
def test_rows(N, C, topk, T, dtype):
    g = torch.Generator().manual_seed(N * 1000 + C)
    x = (torch.randn(N, C, generator=g) * 3).to(DT[dtype])
    y = _labels((N,), C, g, x)
    _run(x.to(DEV), y.to(DEV), topk=topk, temperature=T)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape,topk", [
    ((2049, 1025), 16), ((2100, 1031), 0), ((2051, 2001), 3), ((2048, 4103), 8),       # a wave to a row
    ((2, 30, 257, 257), 8), ((1, 17, 363, 365), 16), ((3, 16, 211, 211), 4),           # a thread to a position
])
def test_many_positions(shape, topk, dtype):
    """Calls that fill the card with one wave to a row, or one thread to a position: with a mask for each row (none,
    one class, half of them left), NaN and infinities where it leaves classes out and in a few rows where it does not."""
    g = torch.Generator().manual_seed(sum(shape))
    N, C = shape[:2]
    x = (torch.randn(shape, generator=g) * 3).to(DT[dtype])
    x[:, C // 3][torch.rand(shape[:1] + shape[2:], generator=g) < 0.01] = math.nan
    x[:, C // 2][torch.rand(shape[:1] + shape[2:], generator=g) < 0.01] = math.inf
    x[:, C - 1][torch.rand(shape[:1] + shape[2:], generator=g) < 0.01] = -math.inf
    y = _labels(shape[:1] + shape[2:], C, g)
    _run(x.to(DEV), y.to(DEV), topk=topk)
    m = _mask(N, C, g)
    x = torch.where(m.view(N, C, *[1] * (len(shape) - 2)), x, torch.full((), math.nan, dtype=x.dtype))
    out, d = _run(x.to(DEV), y.to(DEV), topk=topk, class_mask=m.to(DEV), temperature=0.5)
    assert (out.entropy[0] == 0).all() and (d[0] == 0).all()


def _views(dtype):
    g = torch.Generator().manual_seed(11)
    mk = lambda *s: (torch.randn(*s, generator=g) * 3).to(dtype).to(DEV)  # noqa: E731
    return {
        "crop": (mk(2, 13, 40, 50)[:, :, 3:30, 7:44], 1),
        "crop_even": (mk(2, 16, 40, 64)[:, :, 4:20, 8:40], 1),
        "class_slice": (mk(2, 40, 9, 33)[:, 5:35], 1),
        "every_second_pixel": (mk(2, 13, 20, 50)[:, :, :, ::2], 1),
        "every_second_class": (mk(2, 26, 20, 25)[:, ::2], 1),
        "channels_last": (mk(2, 20, 25, 17).permute(0, 3, 1, 2), 1),
        "nhwc": (mk(2, 9, 11, 30), -1),
        "nhwc_crop": (mk(2, 9, 11, 36)[:, 1:8, 2:9, 3:33], 3),
        "padded_rows": (mk(50, 1040)[:, :1001], 1),
        "padded_rows_offset": (mk(50, 3001)[:, 1:2002], 1),
        "class_first": (mk(30, 500), 0),
        "class_first_narrow": (mk(30, 520)[:, 3:503], 0),
        "class_middle": (mk(3, 5, 17, 4, 6), 2),
        "five_dims_strided": (mk(2, 4, 7, 6, 8, 3)[:, ::2, :, ::2, ::2], 2),
        "expanded": (mk(1, 30, 1, 44).expand(3, 30, 5, 44), 1),
        "one_class_row": (mk(100, 3)[:, 1:2], 1),
        "transposed": (mk(600, 70).t(), 1),
        "transposed_long": (mk(2100, 33).t(), 1),
    }


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("name", sorted(_views(torch.float32)) if torch.cuda.is_available() else ["crop"])
def test_strided_layouts(name, dtype):
    x, dim = _views(DT[dtype])[name]
    g = torch.Generator().manual_seed(5)
    d = dim % x.ndim
    shape = x.shape[:d] + x.shape[d + 1:]
    y = _labels(shape, x.shape[d], g).to(DEV)
    _run(x, y, dim=dim, topk=min(3, x.shape[d]))


def _mask(B, C, gen):
    m = torch.rand(B, C, generator=gen) < 0.5
    m[0] = False                      # a frame without a class
    if B > 1:
        m[1] = False
        m[1, C // 2] = True           # one class alone
    return m


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(4, 30, 9, 13), (3, 128, 16, 64), (5, 19), (4, 1000), (6, 5000), (3, 5, 1)])
@pytest.mark.parametrize("poison", [0.0, math.nan, math.inf, -math.inf])
def test_class_mask_hides_whatever_the_logits_hold(shape, poison, dtype):
    g = torch.Generator().manual_seed(3)
    B, C = shape[:2]
    m = _mask(B, C, g)
    x = (torch.randn(shape, generator=g) * 3).to(DT[dtype])
    x = torch.where(m.view(B, C, *[1] * (len(shape) - 2)), x, torch.full_like(x, poison))
    y = _labels(shape[:1] + shape[2:], C, g)
    out, d = _run(x.to(DEV), y.to(DEV), topk=min(4, C), class_mask=m.to(DEV))
    assert (out.top_ids[0] == -1).all() and (out.entropy[0] == 0).all() and (d[0] == 0).all()
    # one mask for all rows
    m1 = m[2]
    x1 = torch.where(m1.view(1, C, *[1] * (len(shape) - 2)), torch.randn(shape, generator=g).to(DT[dtype]),
                     torch.full((), poison, dtype=DT[dtype]))
    _run(x1.to(DEV), y.to(DEV), topk=min(4, C), class_mask=m1.to(DEV))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("layout", ["planes", "rows", "long_rows"])
def test_degenerate_rows(layout, dtype):
    """-inf, the type's lowest value, NaN, +inf, zeros of both signs, ties, far apart and confident rows."""
    C = {"planes": 37, "rows": 37, "long_rows": 3001}[layout]
    lo = torch.finfo(DT[dtype]).min
    g = torch.Generator().manual_seed(17)
    rows = [torch.randn(C, generator=g) for _ in range(16)]
    rows[0][:] = -math.inf
    rows[1][:] = lo
    rows[2][:] = lo
    rows[2][5] = 1.0
    rows[3][7] = math.nan
    rows[4][9] = math.inf
    rows[5][:] = -math.inf
    rows[5][C - 1] = -2.0
    rows[6][:] = 0.0
    rows[6][1::2] = -0.0
    rows[7][:] = rows[7][:4].repeat(C // 4 + 1)[:C]          # ties
    rows[8][:] *= 100
    rows[9][:] = -90.0
    rows[9][3] = 0.0                                         # nothing left of the others
    rows[10][:] = -17.0
    rows[10][C - 2] = 0.0                                    # confident
    rows[11][:] = torch.arange(C).float() / 8                # the maximum comes last
    rows[12][:] = -torch.arange(C).float() / 8
    rows[13][::3] = -math.inf
    rows[14][4], rows[14][C - 3] = math.nan, math.nan
    rows[15][2], rows[15][C - 5] = math.inf, math.inf
    x = torch.stack(rows).to(DT[dtype])
    y = torch.tensor([0, 1, 5, 3, 9, C - 1, 2, 1, IGN, 3, C - 2, C - 1, C, 0, -1, 2])
    if layout == "planes":
        xx = x.t().contiguous().view(1, C, 4, 4)
        out, d = _run(xx.to(DEV), y.view(1, 4, 4).to(DEV), topk=5)
        ids = out.top_ids.view(5, 16).t()
    else:
        out, d = _run(x.to(DEV), y.to(DEV), topk=5)
        ids = out.top_ids
    assert ids[0].tolist() == [-1] * 5 and ids[5].tolist() == [C - 1, -1, -1, -1, -1]
    assert ids[6].tolist() == [0, 1, 2, 3, 4]                # both zeros are one value
    assert ids[3][0] == 7 and ids[4][0] == 9 and ids[14][:2].tolist() == [4, C - 3]


def test_confident_rows_keep_their_digits():
    """p of the label is 1 - 36 e^-17: -log p and the entropy are small numbers, right to 32 bits, not 0."""
    x = torch.full((1, 37, 8, 8), -17.0)
    x[:, 4] = 0.0
    out = K.label_log_probs(x.to(DEV), torch.full((1, 8, 8), 4).to(DEV))
    r = 36 * math.exp(-17.0)
    want = -math.log1p(r)
    assert abs(out.log_prob[0, 0, 0].item() - want) <= abs(want) * 200 * 2.0 ** -24
    h = math.log1p(r) + 17 * r / (1 + r)
    assert abs(out.entropy[0, 0, 0].item() - h) <= h * 200 * 2.0 ** -24


@pytest.mark.parametrize("layout", ["planes", "rows", "long_rows"])
def test_invalid_labels_are_loud_and_carry_no_gradient(layout):
    C = {"planes": 11, "rows": 11, "long_rows": 2500}[layout]
    g = torch.Generator().manual_seed(2)
    shape = (2, C, 3, 5) if layout == "planes" else (30, C)
    x = torch.randn(shape, generator=g).to(DEV)
    y = torch.randint(0, C, x.shape[:1] + x.shape[2:], generator=g)
    y.view(-1)[[0, 1, 2]] = torch.tensor([-1, C, 1 << 40])
    y.view(-1)[3] = -(1 << 62)
    out = K.label_log_probs(x, y.to(DEV), want_stats=True)
    assert out.log_prob.view(-1)[:4].isnan().all() and out.log_prob.view(-1)[4:].isfinite().all()
    d = K.label_log_probs_bwd(x, out.stats, torch.ones_like(out.log_prob))
    assert (d.movedim(1, -1).reshape(-1, C)[:4] == 0).all()
    # without an ignore label a value like any other is no class either
    out = K.label_log_probs(x, torch.full_like(y, -1).to(DEV), ignore_label=-1)
    assert (out.log_prob == 0).all()


def test_backward_against_differences():
    """The gradient against central differences of the 64-bit operator, and against autograd of it."""
    g = torch.Generator().manual_seed(8)
    x = torch.randn(2, 9, 3, generator=g)
    y = _labels((2, 3), 9, g)
    y[0, 0] = 4
    wl, we = torch.randn(2, 3, generator=g), torch.randn(2, 3, generator=g)

    def f(v):
        o = oracle.label_log_probs(v, y, ignore_label=IGN, temperature=0.8)
        return (o["log_prob"] * wl + o["entropy"] * we).sum()

    xd, h = x.double(), 1e-5
    num = torch.zeros_like(xd)
    for i in range(xd.numel()):
        e = torch.zeros(xd.numel(), dtype=torch.float64)
        e[i] = h
        num.view(-1)[i] = (f(xd + e.view_as(xd)) - f(xd - e.view_as(xd))) / (2 * h)
    a = x.to(DEV).requires_grad_()
    out = ops.label_log_probs(a, y.to(DEV), ignore_label=IGN, temperature=0.8, topk=2)
    (out.log_prob * wl.to(DEV) + out.entropy * we.to(DEV)).sum().backward()
    # differences: h^2 of the third derivative (<= ~10 here) and 2^-52 / h of the value; the kernel: 1e-5 at most
    assert (a.grad.double().cpu() - num).abs().max() < 2e-5


def test_autograd_node():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 30, 9, 8, generator=g).to(DEV)
    y = _labels((2, 9, 8), 30, g).to(DEV)
    # a mean: the gradient that arrives is an expanded scalar; the logits are no leaf and a strided view
    leaf = torch.randn(2, 30, 12, 9, generator=g).to(DEV).requires_grad_()
    out = ops.label_log_probs(leaf[:, :, 2:11, :8] * 2, y, ignore_label=IGN, topk=2)
    assert not out.top_log_probs.requires_grad and not out.top_ids.requires_grad and out.stats is None
    out.log_prob.mean().backward()
    ref = torch.zeros(2, 30, 12, 9, dtype=torch.float64)
    ref[:, :, 2:11, :8] = 2 * oracle.label_log_probs_bwd(leaf.detach()[:, :, 2:11, :8] * 2, y,
                                                         torch.full((2, 9, 8), 1 / 144.0), None, ignore_label=IGN)
    assert (leaf.grad.double().cpu() - ref).abs().max() < 1e-6
    # the entropy alone, without labels; bf16 logits get a bf16 gradient; used twice, the gradients add
    b = x.bfloat16().requires_grad_()
    o1 = ops.label_log_probs(b)
    assert o1.log_prob is None
    (o1.entropy.sum() + ops.label_log_probs(b).entropy.sum()).backward()
    assert b.grad.dtype == torch.bfloat16
    want = 2 * oracle.label_log_probs_bwd(b.detach(), None, None, torch.ones(2, 9, 8))
    # each gradient is rounded to bf16 and so is their sum: 2 x 2^-8 of the value
    assert ((b.grad.double().cpu() - want).abs() <= 2 * 2.0 ** -8 * want.abs() + 1e-5).all()
    # no gradient asked: nothing saved
    assert ops.label_log_probs(x, y).log_prob.grad_fn is None
    with torch.no_grad():
        assert ops.label_log_probs(x.clone().requires_grad_(), y).log_prob.grad_fn is None
    with pytest.raises(RuntimeError):                         # modified between forward and backward
        c = x.clone().requires_grad_()
        z = c * 1
        o = ops.label_log_probs(z, y)
        z.add_(1)
        o.log_prob.sum().backward()


def test_empty_and_same_bits_twice():
    x = torch.zeros(0, 5, 3, device=DEV)
    out = K.label_log_probs(x, torch.zeros(0, 3, dtype=torch.int64, device=DEV), topk=2, want_stats=True)
    assert out.entropy.shape == (0, 3) and out.top_ids.shape == (0, 2, 3)
    assert K.label_log_probs_bwd(x, out.stats, out.log_prob).shape == (0, 5, 3)
    g = torch.Generator().manual_seed(1)
    for shape in ((2, 30, 50, 60), (1, 70001), (300, 5001), (2000, 30)):
        x = torch.randn(shape, generator=g).to(DEV)
        a, b = (K.label_log_probs(x, topk=4) for _ in range(2))
        assert torch.equal(a.entropy, b.entropy) and torch.equal(a.top_log_probs, b.top_log_probs)


def test_offsets_past_32_bits():
    """A class stride and positions past 2^31 elements: bf16 logits of 4.3e9 elements, read at both ends."""
    if torch.cuda.get_device_properties(0).total_memory < 40e9:
        pytest.skip("needs 20 GB")
    big = torch.zeros(3, 2, 720_000_000, dtype=torch.bfloat16, device=DEV)
    cut = big[:, :, -70:]
    g = torch.Generator().manual_seed(0)
    vals = torch.randn(3, 2, 70, generator=g).bfloat16()
    cut.copy_(vals)
    _run(cut, _labels((3, 70), 2, g).to(DEV), topk=2)
    del big, cut
    big = torch.zeros(2_200_000, 1001, dtype=torch.bfloat16, device=DEV)
    cut = big[-3:, :1000]
    cut.copy_(torch.randn(3, 1000, generator=g).bfloat16())
    y = torch.zeros(2_200_000, dtype=torch.int64, device=DEV)
    y[-3:] = torch.tensor([5, 999, 17])
    out = K.label_log_probs(big[:, :1000], y, topk=2)
    ref = oracle.label_log_probs(cut, y[-3:], topk=2)
    assert torch.equal(out.top_ids[-3:].long().cpu(), ref["top_ids"])
    assert (out.log_prob[-3:].double().cpu() - ref["log_prob"]).abs().max() < 1e-3
    assert (out.log_prob[0].item() + math.log(1000)) < 1e-4


def test_streams_and_graphs():
    """On a side stream, and captured: two graphs of different inputs, replayed in turn between eager work."""
    g = torch.Generator().manual_seed(6)
    cases = []
    for shape in ((2, 30, 40, 50), (1, 70001), (64, 300)):
        x = torch.randn(shape, generator=g).to(DEV)
        y = torch.randint(0, shape[1], shape[:1] + shape[2:], generator=g).to(DEV)
        cases.append((x, y, torch.randn(shape[:1] + shape[2:], generator=g).to(DEV)))

    def step(x, y, gl):
        o = K.label_log_probs(x, y, topk=3, want_stats=True)
        return o, K.label_log_probs_bwd(x, o.stats, gl, gl)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = [step(*c) for c in cases]
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for c in cases:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = step(*c)
        graphs.append((gr, res))
    for turn in range(3):
        for i, (x, y, gl) in enumerate(cases):
            x.mul_(1.1)
            graphs[i][0].replay()
            eager, d = step(x, y, gl)
            torch.cuda.synchronize()
            got, gd = graphs[i][1]
            for a, b in zip(got, eager):
                assert torch.equal(a, b)
            assert torch.equal(gd, d)
    for (o, d), c in zip(on_side, cases):
        assert o.log_prob.isfinite().all() and d.isfinite().all()


def test_panoptic_head_reports_entropy_and_alternatives():
    """postprocess_panoptic(alternatives=k): the statistics are those of the head's own logits, the first alternative
    is the label before thresholds, and what it returned before is unchanged."""
    from ldmseg.pipelines.panoptic import postprocess_panoptic
    g = torch.Generator().manual_seed(12)
    lo = (torch.randn(2, 19, 12, 20, generator=g) * 4).to(DEV)
    pad = torch.zeros(2, 48, 80, dtype=torch.bool, device=DEV)
    pad[:, :41, 3:77] = True
    args = (lo, (48, 80), pad, [(83, 147), (41, 74)], 0.5, 20, 0.5, 255)
    plain = postprocess_panoptic(*args)
    more = postprocess_panoptic(*args, alternatives=3)
    bare = postprocess_panoptic(*args, alternatives=0)
    for i, (a, b, c) in enumerate(zip(plain, more, bare)):
        assert set(a) == {"panoptic_seg", "cleaned_pred"} and set(c) == set(a) | {"entropy"}
        assert torch.equal(a["cleaned_pred"], b["cleaned_pred"]) and torch.equal(b["entropy"], c["entropy"])
        assert torch.equal(a["panoptic_seg"][0], b["panoptic_seg"][0])
        m = K.resize_bilinear(lo, size=(48, 80))[i:i + 1, :, :41, 3:77]
        m = K.resize_bilinear(m, size=args[3][i])
        ref = oracle.label_log_probs(m, topk=3)
        ids, lp = b["alternatives"]
        assert torch.equal(ids.long().cpu(), ref["top_ids"][0])
        assert (lp.double().cpu() - ref["top_log_probs"][0]).abs().max() < 2e-5
        assert (b["entropy"].double().cpu() - ref["entropy"][0]).abs().max() < 2e-5
        kept = b["cleaned_pred"] >= 0
        assert torch.equal(b["cleaned_pred"][kept], ids[0].long()[kept])


def test_training_step_of_both_operators():
    """Loss, gradient, norm and clip together, as a training loop uses them: a small head on bf16 features, its loss the
    labels' log probability and an entropy term, two steps of SGD; against the same in 64 bits."""
    from ldmseg.trainers import clip_grad_norm_
    g = torch.Generator().manual_seed(21)
    B, D, C, H, W, limit, lr = 3, 16, 30, 17, 23, 0.05, 0.5
    feats = torch.randn(B, D, H, W, generator=g)
    y = _labels((B, H, W), C, g)
    y[0, 0, :3] = 7
    w0, b0 = torch.randn(C, D, generator=g) * 0.3, torch.randn(C, generator=g) * 0.1
    n = (y != IGN).sum().item()

    head = torch.nn.Conv2d(D, C, 1).to(DEV)
    with torch.no_grad():
        head.weight.copy_(w0.view(C, D, 1, 1))
        head.bias.copy_(b0)
    rw, rb = w0.double().requires_grad_(), b0.double().requires_grad_()
    x, yd = feats.to(DEV), y.to(DEV)
    for step in range(2):
        logits = torch.nn.functional.conv2d(x, head.weight, head.bias)
        out = ops.label_log_probs(logits, yd, ignore_label=IGN)
        (-out.log_prob.sum() / n - 0.01 * out.entropy.mean()).backward()
        norm = clip_grad_norm_(head.parameters(), limit)

        z = torch.einsum("bdhw,cd->bchw", feats.double(), rw) + rb.view(1, C, 1, 1)
        lp = torch.log_softmax(z, 1)
        ent = -(lp.exp() * lp).sum(1)
        nll = -lp.gather(1, y.clamp(max=C - 1)[:, None])[:, 0][y != IGN].sum() / n
        gw, gb = torch.autograd.grad(nll - 0.01 * ent.mean(), (rw, rb))
        rn = torch.sqrt(gw.square().sum() + gb.square().sum())
        assert rn > limit and abs(norm.item() - rn.item()) < 1e-4 * rn.item()
        f = limit / (rn + 1e-6)
        # fp32 products of 16 terms and sums of 1173 positions in torch's convolution: a few 1e-5 relative to the norm
        assert (head.weight.grad.view(C, D).double().cpu() - gw * f).abs().max() < 1e-4 * limit
        assert (head.bias.grad.double().cpu() - gb * f).abs().max() < 1e-4 * limit
        with torch.no_grad():
            for p in head.parameters():
                p.sub_(p.grad, alpha=lr)
                p.grad = None
            rw -= lr * f * gw
            rb -= lr * f * gb


def test_clipping_the_drop_in_unet():
    """loss.backward() through the drop-in UNet's autograd node leaves one fp32 tensor per parameter: clip_grad_norm_
    clips them as torch's own does."""
    from ldmseg.models import UNet
    from ldmseg.trainers import clip_grad_norm_
    torch.manual_seed(0)
    u = UNet(block_out_channels=(64, 128, 128, 128), cross_attention_dim=None)
    u.modify_encoder(in_channels=8, init_mode_seg="copy", init_mode_image="random")
    u.freeze_layers(["time_embedding"])
    u = u.to(DEV).train()
    out = u(torch.randn(1, 8, 16, 16, device=DEV), torch.tensor([500], device=DEV)).sample
    out.square().mean().backward()
    ps = [p for p in u.parameters() if p.grad is not None]
    assert len(ps) > 200
    twin = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, q in zip(ps, twin):
        q.grad = p.grad.clone()
    nt = torch.nn.utils.clip_grad_norm_(twin, 1e-3)
    n = clip_grad_norm_(u.parameters(), 1e-3)
    assert n > 1e-3 and abs(n.item() - nt.item()) <= 1e-5 * nt.item()
    for p, q in zip(ps, twin):
        torch.testing.assert_close(p.grad, q.grad, rtol=2e-5, atol=0)
    assert abs(K.grad_norm([p.grad for p in ps]).item() - 1e-3) < 1e-6


def test_mask_rows_that_do_not_divide_the_positions():
    """The C entry takes any number of positions to a mask row: the last row's may be fewer, and nothing behind the
    last position is written."""
    import ctypes
    g = torch.Generator().manual_seed(9)
    C, N, div = 20, 330, 128                        # rows of 128, 128 and 74 positions
    x = torch.randn(C, N, generator=g).to(DEV)
    m = (torch.rand(3, C, generator=g) < 0.5).to(DEV)
    m[:, 3] = True
    ent, stats = torch.full((N + 300,), 7.0, device=DEV), torch.full((4 * N + 300,), 7.0, device=DEV)
    d = torch.full((C * N + 300,), 7.0, device=DEV)
    ge = torch.randn(N, generator=g).to(DEV)
    lib, st = K.load_library(), torch.cuda.current_stream().cuda_stream
    common = dict(logits=x.data_ptr(), n0=1, n1=1, n2=N, s2=1, classes=C, sc=N, class_mask=m.data_ptr(), mask_stride=C,
                  mask_div=div, temperature=1.0, dtype=0)
    p = K.LabelProbsParams(**common, inner=N, entropy=ent.data_ptr(), stats=stats.data_ptr())
    assert lib.ldm_label_log_probs(ctypes.byref(p), st) == 0
    b = K.LabelProbsBwdParams(**common, stats=stats.data_ptr(), d_entropy=ge.data_ptr(), d_logits=d.data_ptr(), o2=1, oc=N)
    assert lib.ldm_label_log_probs_bwd(ctypes.byref(b), st) == 0
    for r in range(3):
        s = slice(r * div, min(N, (r + 1) * div))
        ref = oracle.label_log_probs(x[:, s], dim=0, class_mask=m[r])
        assert (ent[s].double().cpu() - ref["entropy"]).abs().max() < 1e-5
        want = oracle.label_log_probs_bwd(x[:, s], None, None, ge[s], dim=0, class_mask=m[r])
        assert (d[:C * N].view(C, N)[:, s].double().cpu() - want).abs().max() < 1e-5
    assert (ent[N:] == 7).all() and (stats[4 * N:] == 7).all() and (d[C * N:] == 7).all()
