"""Label probabilities and gradient clipping without a GPU: refusals, the layout of strided positions, and the 64-bit
restatement against torch's own log_softmax."""
import math

import pytest
import torch

from ldmseg.ops import native as K
from ldmseg.trainers import clip_grad_norm_
from oracle import label_probs as oracle

ERR_OVERLAP = 4


def _refuses(exc, match, *a, **kw):
    with pytest.raises(exc, match=match):
        K.label_log_probs(*a, **kw)


def test_label_log_probs_refusals():
    x, y = torch.zeros(2, 5, 3, 4), torch.zeros(2, 3, 4, dtype=torch.int64)
    _refuses(RuntimeError, "GPU tensors only", x, y)
    _refuses(TypeError, "unsupported dtype", x.half(), y)
    _refuses(TypeError, "unsupported dtype", x.double(), y)
    _refuses(TypeError, "int64", x, y.int())
    _refuses(ValueError, "labels must be", x, y[:1])
    _refuses(ValueError, "labels must be", x, y, dim=2)
    _refuses(ValueError, "outside", x, dim=4)
    _refuses(ValueError, "outside", x, dim=-5)
    _refuses(ValueError, "class dim and at least", torch.zeros(4))
    _refuses(ValueError, "no classes", torch.zeros(2, 0, 3))
    _refuses(ValueError, "topk", x, topk=6)
    _refuses(ValueError, "topk", x, topk=-1)
    _refuses(ValueError, "topk", torch.zeros(2, 50), topk=17)
    for t in (0.0, -1.0, 1e-5, 1e5, math.nan, math.inf):
        _refuses(ValueError, "temperature", x, temperature=t)
    _refuses(TypeError, "class_mask", x, class_mask=torch.ones(5))
    _refuses(ValueError, "class_mask must be", x, class_mask=torch.ones(3, 5, dtype=torch.bool))
    _refuses(ValueError, "class_mask must be", x, class_mask=torch.ones(4, dtype=torch.bool))
    _refuses(ValueError, "class_mask must be", torch.zeros(5, 2), dim=0,
             class_mask=torch.ones(5, 5, dtype=torch.bool))


def test_label_log_probs_bwd_refusals():
    x, s, g = torch.zeros(2, 5, 3), torch.zeros(4, 2, 3), torch.zeros(2, 3)

    def refuses(exc, match, *a, **kw):
        with pytest.raises(exc, match=match):
            K.label_log_probs_bwd(*a, **kw)

    refuses(RuntimeError, "GPU tensors only", x, s, g, g)
    refuses(ValueError, "stats", x, s[:3], g)
    refuses(ValueError, "stats", x, s.double(), g)
    refuses(ValueError, "stats", x, s.transpose(1, 2).contiguous().transpose(1, 2), g)
    refuses(ValueError, "d_log_prob", x, s, g.double())
    refuses(ValueError, "d_log_prob", x, s, g[:1])
    refuses(ValueError, "d_entropy", x, s, None, g.view(-1))
    refuses(ValueError, "temperature", x, s, g, temperature=0.0)
    refuses(TypeError, "unsupported dtype", x.half(), s, g)


def test_c_entries_refuse_before_any_launch():
    """The C entry checks what the Python layer would never send; nothing is launched without a GPU."""
    import ctypes
    lib = K.load_library()
    ok = dict(n0=1, n1=1, n2=4, s2=1, classes=5, sc=4, inner=4, temperature=1.0, dtype=0, logits=16, entropy=16)
    for bad in (dict(classes=0), dict(classes=1 << 31), dict(n2=-1), dict(n1=1 << 39), dict(s2=-1), dict(sc=-4),
                dict(temperature=0.0), dict(temperature=math.nan), dict(dtype=2), dict(topk=17), dict(topk=6),
                dict(topk=2), dict(logits=None), dict(entropy=None), dict(labels=16), dict(inner=3), dict(inner=0),
                dict(class_mask=16, mask_div=0), dict(class_mask=16, mask_div=4, mask_stride=-1)):
        p = K.LabelProbsParams(**{**ok, **bad})
        assert lib.ldm_label_log_probs(ctypes.byref(p), None) == 1, bad
    for big in (dict(n2=1 << 32, inner=(1 << 32) + 256), dict(n2=1 << 26, sc=1, s2=600, classes=600, inner=1),
                dict(n2=1 << 24, sc=1, s2=9000, classes=9000, inner=1), dict(n2=1 << 27, sc=1, s2=3000, classes=3000, inner=1)):
        assert lib.ldm_label_log_probs(ctypes.byref(K.LabelProbsParams(**{**ok, **big, "n2": big["n2"] + 256})), None) == 1
    assert lib.ldm_label_log_probs(None, None) == 1
    assert lib.ldm_label_log_probs(ctypes.byref(K.LabelProbsParams(**{**ok, "n2": 0})), None) == 0
    okb = dict(n0=1, n1=1, n2=4, s2=1, classes=5, sc=4, o2=1, oc=4, temperature=1.0, dtype=0, logits=16, stats=16,
               d_logits=16)
    for bad in (dict(classes=-1), dict(o2=-1), dict(oc=-1), dict(stats=None), dict(d_logits=None), dict(logits=None),
                dict(dtype=7), dict(temperature=-1.0), dict(class_mask=16, mask_div=0)):
        p = K.LabelProbsBwdParams(**{**okb, **bad})
        assert lib.ldm_label_log_probs_bwd(ctypes.byref(p), None) == 1, bad
    u64, i64 = ctypes.c_uint64, ctypes.c_int64
    ptrs, numel = (u64 * 2)(4096, 1 << 20), (i64 * 2)(16, 65536)
    assert lib.ldm_grad_norm_workspace_bytes((i64 * 2)(16, 16), 2) == 0      # one block takes no partials
    wsb = lib.ldm_grad_norm_workspace_bytes(numel, 2)
    assert wsb > 0

    def norm(ptrs=ptrs, numel=numel, codes=b"\0\0", n=2, kind=0, limit=1.0, clip=1, out=64, ws=64, wsb=wsb):
        return lib.ldm_grad_norm(ptrs, numel, codes, n, kind, limit, clip, out, ws, wsb, None)

    assert norm(ptrs=(u64 * 2)(4096, 4096)) == norm(ptrs=(u64 * 2)(4096, 4156)) == ERR_OVERLAP
    assert "overlap" in lib.ldm_status_string(ERR_OVERLAP).decode()
    for kw in (dict(ptrs=(u64 * 2)(0, 1 << 20)),
               dict(numel=(i64 * 2)(-1, 16)), dict(codes=b"\0\2"), dict(n=0), dict(n=-1), dict(kind=3), dict(kind=-1),
               dict(limit=-1.0), dict(limit=math.nan), dict(clip=3), dict(clip=-1), dict(out=None), dict(ws=None),
               dict(wsb=wsb - 1), dict(ptrs=None), dict(ptrs=(u64 * 2)(1 << 63, 1 << 20))):
        assert norm(**kw) == 1, kw
    assert norm(ptrs=(u64 * 2)(4098, 1 << 20)) == 2          # fp32 at a 2-byte address
    assert norm(ptrs=(u64 * 2)(4097, 1 << 20), codes=b"\1\0") == 2


def test_clip_refusals():
    p = torch.nn.Parameter(torch.zeros(4))
    assert clip_grad_norm_([p], 1.0) == 0                     # no gradients
    assert clip_grad_norm_(p, 1.0) == 0 and clip_grad_norm_(iter([]), 1.0) == 0
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        clip_grad_norm_([p], 1.0)
    for bad in (3.0, 0.0, -math.inf, math.nan):
        with pytest.raises(ValueError, match="norm_type"):
            clip_grad_norm_([p], 1.0, norm_type=bad)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_([p], bad)
    q = torch.nn.Parameter(torch.zeros(4, dtype=torch.float16))
    q.grad = torch.ones(4, dtype=torch.float16)
    with pytest.raises(TypeError, match="unsupported gradient dtype"):
        clip_grad_norm_([p, q], 1.0)
    for bad in (torch.ones(1).expand(4), torch.ones(8)[::2]):
        with pytest.raises(ValueError, match="dense"):
            K.grad_norm([bad])
    with pytest.raises(TypeError, match="sparse"):
        K.grad_norm([torch.ones(4).to_sparse()])
    with pytest.raises(TypeError, match="must be a tensor"):
        K.grad_norm([torch.ones(4), 3])
    with pytest.raises(TypeError, match="iterable"):
        K.grad_norm(7)
    for dense in (torch.zeros(2, 3, 4, 5).permute(0, 2, 3, 1), torch.zeros(3, 0, 2), torch.zeros(()),
                  torch.zeros(5, 1).expand(5, 1)):
        with pytest.raises(RuntimeError, match="GPU tensors only"):      # dense in any order: only the device is wrong
            K.grad_norm([dense])


@pytest.mark.parametrize("make,dim", [
    (lambda x: x, 1), (lambda x: x[:, :, 1:4, 2:6], 1), (lambda x: x.permute(0, 2, 3, 1), 3),
    (lambda x: x.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2), 1), (lambda x: x[:, ::2, :, ::3], 1),
    (lambda x: x[:, :, 1:2], 1), (lambda x: x, 0), (lambda x: x, -1), (lambda x: x[:1].expand(3, 5, 6, 8), 1),
    (lambda x: x.permute(3, 1, 0, 2), 1), (lambda x: x.unflatten(3, (2, 2, 2)).permute(4, 0, 2, 1, 3, 5), 3),
])
def test_strided_positions_address_every_element(make, dim):
    """Walking the merged sizes and strides visits x, and the gradient's tensor, in the order of the labels."""
    base = torch.arange(2 * 5 * 6 * 8).view(2, 5, 6, 8)
    x = make(base)
    dim = dim % x.ndim
    y, n, s, inner, out, o = K.torch_binding().label_positions(x, dim)
    N = n[0] * n[1] * n[2]
    idx = [torch.arange(k) for k in n]
    grid = sum(i.view([-1 if j == d else 1 for j in range(3)]) * st for d, (i, st) in enumerate(zip(idx, s)))
    want = x.movedim(dim, 0).reshape(x.shape[dim], -1)
    flat = torch.as_strided(y, (y.untyped_storage().size() // y.element_size(),), (1,), 0)
    for c in range(x.shape[dim]):
        at = y.storage_offset() + grid.reshape(-1) + c * y.stride(dim)
        assert torch.equal(flat[at], want[c])
    assert N == want.shape[1] and N % inner == 0
    out.copy_(x)
    grid = sum(i.view([-1 if j == d else 1 for j in range(3)]) * st for d, (i, st) in enumerate(zip(idx, o)))
    flat = torch.as_strided(out, (out.untyped_storage().size() // out.element_size(),), (1,), 0)
    for c in range(x.shape[dim]):
        assert torch.equal(flat[grid.reshape(-1) + c * out.stride(dim)], want[c])


def test_oracle_is_log_softmax():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 7, 5, generator=g).double().requires_grad_()
    y = torch.randint(0, 7, (3, 5), generator=g)
    o = oracle.label_log_probs(x, y, topk=3, temperature=0.6)
    lp = torch.log_softmax(x / 0.6, 1)
    torch.testing.assert_close(o["log_prob"], lp.gather(1, y[:, None])[:, 0].detach())
    h = -(lp.exp() * lp).sum(1)
    torch.testing.assert_close(o["entropy"], h.detach())
    torch.testing.assert_close(o["top_log_probs"], lp.topk(3, 1).values.detach())
    wl, we = torch.randn(3, 5, generator=g).double(), torch.randn(3, 5, generator=g).double()
    (lp.gather(1, y[:, None])[:, 0] * wl + h * we).sum().backward()
    torch.testing.assert_close(oracle.label_log_probs_bwd(x, y, wl, we, temperature=0.6), x.grad)
    nan = oracle.label_log_probs(torch.tensor([[1.0, math.nan, 2.0], [math.inf, 0.0, 1.0], [-math.inf] * 3]), topk=2)
    assert nan["entropy"][:2].isnan().all() and nan["entropy"][2] == 0
    assert nan["top_ids"].tolist() == [[1, 2], [0, 2], [-1, -1]]
