"""Global gradient norm over many tensors and clipping on the HIP path (ldm_grad_norm), against 64 bits and against
torch.nn.utils.clip_grad_norm_.

Tolerances: the sums are fp64 and the norm is rounded once to fp32 (2^-24).  The factor rounds in norm + 1e-6, in the
division, and inherits the norm's and the limit's rounding: 4 x 2^-24; its product with a gradient rounds once more: an
fp32 gradient is within 5 x 2^-24 relative of the exact one (and 2^-149 where the product is subnormal).  A bf16 gradient
is multiplied by the factor in bf16 and rounded: 2 x 2^-8 + 2^-16 + 4 x 2^-24 (and 2^-134)."""
import math

import pytest
import torch

from ldmseg.ops import native as K
from ldmseg.trainers import clip_grad_norm_

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _params(sizes, dtypes, gen, scale=1.0):
    ps = []
    for i, n in enumerate(sizes):
        dt = dtypes[i % len(dtypes)]
        p = torch.nn.Parameter(torch.zeros(n, dtype=dt, device=DEV))
        p.grad = (torch.randn(n, generator=gen) * scale).to(dt).to(DEV)
        ps.append(p)
    return ps


def _norm(grads, kind):
    parts = [torch.linalg.vector_norm(g.double(), kind) for g in grads if g.numel()]
    return torch.linalg.vector_norm(torch.stack(parts), kind).item() if parts else 0.0


def _check(params, max_norm, kind=2.0):
    before = [p.grad.clone() for p in params]
    want = _norm(before, kind)
    got = clip_grad_norm_(params, max_norm, norm_type=kind)
    assert got.dtype == torch.float32 and got.ndim == 0 and got.is_cuda
    assert abs(got.item() - want) <= 1.01 * U * want
    f = min(1.0, max_norm / (want + 1e-6))
    for p, b in zip(params, before):
        if f == 1.0:
            assert torch.equal(p.grad, b)
            continue
        exact = b.double() * f
        rel = 5.02 * U if b.dtype == torch.float32 else 2.0 ** -7 + 2.0 ** -16 + 5 * U
        tiny = 2.0 ** -149 if b.dtype == torch.float32 else 2.0 ** -134
        assert ((p.grad.double() - exact).abs() <= rel * exact.abs() + tiny).all()


SIZES = {
    "one": [1], "two": [2], "odd": [3, 1, 7, 63, 65], "edges": [255, 256, 257, 8191, 8192, 8193],
    "many": [1 + (i * 37) % 301 for i in range(700)], "table_full": [5] * 224, "table_over": [5] * 225,
    "listed_long": [40_001] * 300, "large": [3_000_001, 17, 2_097_152, 0, 9], "zero_sized": [0, 4, 0], "only_zero_sized": [0, 0],
    "around_one_block": [16_384, 16_383, 1], "around_one_block_over": [32_768, 1, 32_769],
}


@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.bfloat16, torch.float32]],
                         ids=["fp32", "bf16", "mixed"])
@pytest.mark.parametrize("kind", [2.0, math.inf, 1.0], ids=["2", "inf", "1"])
@pytest.mark.parametrize("name", sorted(SIZES))
def test_clip_against_64_bits(name, kind, dtypes):
    g = torch.Generator().manual_seed(len(name))
    ps = _params(SIZES[name], dtypes, g)
    total = _norm([p.grad for p in ps], kind)
    _check(ps, total * 2 + 1, kind)          # within the limit: untouched
    _check(ps, total * 0.37, kind)           # over it
    assert abs(K.grad_norm([p.grad for p in ps], kind).item() - _norm([p.grad for p in ps], kind)) \
        <= 1.01 * U * total
    _check(ps, 0.0, kind)


def test_misaligned_views_of_a_bucket():
    """Gradients as views of one buffer at every element offset (data-parallel buckets), each type; the gaps
    between them stay as they were."""
    for dtype in (torch.float32, torch.bfloat16):
        g = torch.Generator().manual_seed(3)
        flat = torch.randn(100_000, generator=g).to(dtype).to(DEV)
        kept = flat.clone()
        ps, at, used = [], 1, torch.zeros(100_000, dtype=torch.bool)
        for n in (1, 2, 3, 5, 8, 13, 100, 1000, 1001, 4099, 8191, 30_001, 20_000):
            p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device=DEV))
            p.grad = flat[at:at + n]
            used[at:at + n] = True
            ps.append(p)
            at += n + (n % 3)
        _check(ps, 10.0)
        assert torch.equal(flat.cpu()[~used], kept.cpu()[~used])


def test_dense_orders_and_shapes():
    g = torch.Generator().manual_seed(5)
    conv = torch.nn.Parameter(torch.zeros(8, 6, 3, 3, device=DEV).to(memory_format=torch.channels_last))
    conv.grad = torch.randn(8, 6, 3, 3, generator=g).to(DEV).to(memory_format=torch.channels_last)
    lin = torch.nn.Parameter(torch.zeros(5, 7, device=DEV).t())
    lin.grad = torch.randn(5, 7, generator=g).to(DEV).t()
    scalar = torch.nn.Parameter(torch.zeros((), device=DEV))
    scalar.grad = torch.randn((), generator=g).to(DEV)
    none = torch.nn.Parameter(torch.zeros(3, device=DEV))
    _check([conv, lin, scalar], 0.5)
    assert clip_grad_norm_([none, conv], 1e9) > 0 and none.grad is None
    assert clip_grad_norm_(conv, 1e9) > 0
    assert clip_grad_norm_((p for p in [conv, lin]), 1e9) > 0


def test_matches_torch():
    g = torch.Generator().manual_seed(9)
    for kind in (2.0, math.inf, 1.0):           # fp32: of bf16 gradients torch holds the norm itself in bf16
        a = _params(SIZES["many"], [torch.float32], g)
        b = [torch.nn.Parameter(p.detach().clone()) for p in a]
        for p, q in zip(a, b):
            q.grad = p.grad.clone()
        na = clip_grad_norm_(a, 1.5, kind)
        nb = torch.nn.utils.clip_grad_norm_(b, 1.5, kind)
        assert abs(na.item() - nb.item()) <= 1e-5 * nb.item()      # torch sums in fp32
        for p, q in zip(a, b):
            torch.testing.assert_close(p.grad, q.grad, rtol=2e-5, atol=0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_non_finite_and_extreme_values(dtype):
    def grads(*values):
        ps = [torch.nn.Parameter(torch.zeros(5, dtype=dtype, device=DEV)) for _ in values]
        for p, v in zip(ps, values):
            p.grad = torch.full((5,), v, dtype=dtype, device=DEV)
        return ps

    for kind in (2.0, math.inf, 1.0):
        for bad in (math.inf, -math.inf, math.nan):
            ps = grads(1.0, bad, 2.0)
            with pytest.raises(RuntimeError, match="not finite"):
                clip_grad_norm_(ps, 1.0, kind, error_if_nonfinite=True)
            assert (ps[0].grad == 1).all()                          # nothing was scaled
            n = clip_grad_norm_(ps, 1.0, kind)
            qs = grads(1.0, bad, 2.0)
            m = torch.nn.utils.clip_grad_norm_(qs, 1.0, kind)
            assert torch.equal(n.isnan(), m.isnan()) and (n.isnan() or n == m)
            for p, q in zip(ps, qs):
                torch.testing.assert_close(p.grad, q.grad, rtol=0, atol=0, equal_nan=True)
    # squares that leave fp32 on either side do not leave fp64
    for v in (1e30, 1e-30):
        ps = grads(v, v)
        x = ps[0].grad[0].double().item()
        n = clip_grad_norm_(ps, 1e-32)
        assert abs(n.item() - x * math.sqrt(10)) <= 1.01 * U * x * math.sqrt(10)
    assert grads(1e30)[0].grad.isfinite().all()
    ps = grads(2.0)
    assert clip_grad_norm_(ps, 1e9, error_if_nonfinite=True) > 4
    ps = grads(2.0)
    n = clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
    assert abs(n.item() - 2 * math.sqrt(5)) < 1e-6
    assert abs(ps[0].grad.float().norm().item() - 1.0) < 1e-2
    # all zeros: the norm is 0, the factor 1
    ps = grads(0.0)
    assert clip_grad_norm_(ps, 1.0) == 0 and (ps[0].grad == 0).all()


def test_clipping_is_seen_by_autograd():
    """A gradient that a graph has saved is modified in place: the graph's backward refuses, as after torch's clip."""
    p = torch.nn.Parameter(torch.ones(4, device=DEV))
    p.grad = torch.full((4,), 3.0, device=DEV)
    w = torch.ones(4, device=DEV, requires_grad=True)
    y = (w * p.grad).sum()
    assert abs(K.grad_norm(p.grad).item() - 6.0) < 1e-6        # a tensor alone is a list of one; reading changes nothing
    clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        q = torch.ones(3, device=DEV)
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        K.clip_grads([q], 1.0)
    assert (q == 1).all()


def test_a_gradient_listed_twice_is_refused():
    p = torch.nn.Parameter(torch.zeros(100, device=DEV))
    p.grad = torch.ones(100, device=DEV)
    q = torch.nn.Parameter(torch.zeros(60, device=DEV))
    q.grad = p.grad[40:]
    for ps in ([p, p], [p, q], [q, p]):
        with pytest.raises(ValueError, match="overlap"):
            clip_grad_norm_(ps, 1.0)
    assert (p.grad == 1).all()
    p.grad = torch.ones(1, device=DEV).expand(100)
    with pytest.raises(ValueError, match="dense"):
        clip_grad_norm_([p], 1.0)
    p.grad = torch.ones(100, device="cpu").to(DEV)
    c = torch.nn.Parameter(torch.zeros(3))
    c.grad = torch.ones(3)
    with pytest.raises(ValueError, match="one device"):
        clip_grad_norm_([p, c], 1.0)


def test_same_bits_twice_and_on_a_side_stream():
    g = torch.Generator().manual_seed(1)
    ps = _params([100_003, 5, 3_000_001, 77] * 60, [torch.float32, torch.bfloat16], g)
    grads = [p.grad for p in ps]
    a = K.grad_norm(grads)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = K.grad_norm(grads)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b) and torch.equal(a, K.grad_norm(grads))


def test_graph_replays():
    """Captured clipping of two parameter sets, replayed in turn between eager work: the table of addresses is the
    graph's own, and every replay clips what the gradients hold by then."""
    g = torch.Generator().manual_seed(2)
    sets = [_params(SIZES["many"], [torch.float32, torch.bfloat16], g), _params([1000, 3], [torch.float32], g),
            _params([5_000_000, 1_000_003], [torch.float32], g)]
    graphs = []
    for ps in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            n = clip_grad_norm_(ps, 1.0)
        graphs.append((gr, n))
    for turn in range(3):
        for ps, (gr, n) in zip(sets, graphs):
            for p in ps:
                p.grad.normal_(0, 0.5 + turn)
            twin = [torch.nn.Parameter(p.detach().clone()) for p in ps]
            for p, q in zip(ps, twin):
                q.grad = p.grad.clone()
            m = clip_grad_norm_(twin, 1.0)
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(n, m)
            for p, q in zip(ps, twin):
                assert torch.equal(p.grad, q.grad)


def test_large_tensor_in_pieces():
    """One bf16 gradient above 2^31 elements: listed in pieces, indexed in 64 bits."""
    n = (1 << 31) + 12_345
    p = torch.nn.Parameter(torch.empty(n, dtype=torch.bfloat16, device=DEV))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    p.grad[-3:] = 4.0
    p.grad[:1] = 3.0
    p.grad[(1 << 30) - 1:(1 << 30) + 1] = 2.0
    want = math.sqrt(9 + 8 + 48)
    got = clip_grad_norm_([p], want / 2)
    assert abs(got.item() - want) < 1e-5
    assert p.grad[-1] == 2.0 and p.grad[0] == 1.5 and p.grad[1 << 30] == 1.0 and p.grad[5] == 0
