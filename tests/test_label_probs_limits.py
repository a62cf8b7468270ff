"""Sizes at the limits of the label-probability and gradient-norm C entries: what is refused, and what reaches the
launch.  Addresses are made up, so these run only where there is no GPU to launch on."""
import ctypes

import pytest
import torch

from ldmseg.ops import native as K

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses must never be launched on")
OK, ERR_ARG, ERR_LAUNCH = 0, 1, 3


def _fwd(**kw):
    p = K.LabelProbsParams(**{**dict(n0=1, n1=1, n2=4, s2=1, classes=5, sc=4, inner=1, temperature=1.0, dtype=0,
                                     logits=16, entropy=16), **kw})
    lib = K.load_library()
    return lib.ldm_label_log_probs(ctypes.byref(p), None), lib.ldm_label_log_probs_workspace_bytes(ctypes.byref(p))


def _bwd(**kw):
    p = K.LabelProbsBwdParams(**{**dict(n0=1, n1=1, n2=4, s2=1, classes=5, sc=4, o2=1, oc=4, temperature=1.0, dtype=0,
                                        logits=16, stats=16, d_logits=16), **kw})
    return K.load_library().ldm_label_log_probs_bwd(ctypes.byref(p), None)


@pytest.mark.parametrize("n", [
    (1 << 32, 1 << 32, 1), (1 << 22, 1 << 22, 1 << 22), (3, 6148914691236517206, 1), (1, 1 << 62, 6), (1 << 39, 1, 1),
    (1, 1 << 39, 1), (1 << 13, 1 << 13, 1 << 13)])
def test_a_product_of_positions_past_64_bits_is_refused(n):
    """2^32 x 2^32 is 0 in 64 bits and 3 x 6148914691236517206 is 2: neither is a call of that many positions."""
    kw = dict(n0=n[0], n1=n[1], n2=n[2])
    for layout in (dict(), dict(sc=1, s2=600, classes=600, oc=1, o2=600), dict(sc=1, s2=70000, classes=70000, oc=1, o2=70000)):
        fwd = {k: v for k, v in layout.items() if k not in ("oc", "o2")}
        assert _fwd(**kw, **fwd) == (ERR_ARG, 0), layout
        assert _bwd(**kw, **layout) == ERR_ARG, layout
    assert _fwd()[0] == ERR_LAUNCH and _bwd() == ERR_LAUNCH          # what is accepted reaches the launch
    assert _fwd(n0=0)[0] == OK and _bwd(n1=0) == OK


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("n", [1, 2, 32, 63, 64, 127, 128, 100_000])
@pytest.mark.parametrize("classes", [16, 524_280, 524_281, 600_000, 1 << 20, (1 << 21) - 1, 1 << 21])
def test_the_backward_takes_the_strided_classes_that_the_forward_takes(classes, n, dtype):
    kw = dict(n2=n, classes=classes, sc=n + 1, dtype=dtype)
    assert _fwd(**kw)[0] == ERR_LAUNCH
    assert _bwd(**kw, oc=n + 1) == ERR_LAUNCH
    mask = dict(class_mask=16, mask_stride=classes, mask_div=n)
    assert _bwd(**kw, **mask, oc=n + 1) == ERR_LAUNCH


@pytest.mark.parametrize("dtype", [0, 1])
def test_the_documented_limits(dtype):
    """At the limit a call reaches the launch, one more is refused."""
    def rows(classes, n):
        kw = dict(n2=n, classes=classes, sc=1, s2=classes, dtype=dtype, workspace=16, workspace_bytes=1 << 40)
        return _fwd(**kw)[0]

    def rows_bwd(classes, n):
        return _bwd(n2=n, classes=classes, sc=1, s2=classes, oc=1, o2=classes, dtype=dtype)

    top = (1 << 32) - 256
    planes = dict(classes=5, s2=5, sc=2, dtype=dtype)
    assert _fwd(n2=top, **planes)[0] == ERR_LAUNCH and _fwd(n2=top + 1, **planes)[0] == ERR_ARG
    assert _bwd(n2=top, o2=5, oc=2, **planes) == ERR_LAUNCH and _bwd(n2=top + 1, o2=5, oc=2, **planes) == ERR_ARG
    for n in (1, 64, 100_000):
        assert _bwd(n2=n, classes=(1 << 21) + 1, sc=n + 1, oc=n + 1, dtype=dtype) == ERR_ARG
    assert rows(8193, (1 << 24) - 1) == ERR_LAUNCH and rows(8193, 1 << 24) == ERR_ARG
    for classes in (8, 100, 1024, 1025, 8192):
        assert rows(classes, (1 << 25) - 4) == ERR_LAUNCH
    run = 4096 // (2 if dtype else 4)
    assert rows_bwd(run, (1 << 24) - 1) == ERR_LAUNCH and rows_bwd(run, 1 << 24) == ERR_ARG
    assert rows_bwd(run // 256, top) == ERR_LAUNCH and rows_bwd(run // 256, top + 1) == ERR_ARG


@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("numel", [[1 << 62], [(1 << 62) + 5], [(1 << 63) - 1], [1 << 61, 7], [(1 << 46) + 1],
                                   [1 << 45] * 3, [16, (1 << 63) - 8, 16]])
def test_gradients_past_the_address_space_are_refused(numel, code):
    """2^62 fp32 values are 0 bytes in 64 bits and 2^62 + 5 are 20: a clip of them must not answer that all is well."""
    lib = K.load_library()
    n = len(numel)
    sizes, codes = (ctypes.c_int64 * n)(*numel), bytes([code]) * n
    ptrs = (ctypes.c_uint64 * n)(*[4096 + (i << 55) for i in range(n)])
    assert lib.ldm_grad_norm_workspace_bytes(sizes, n) == 0
    for clip in (0, 1, 2):
        assert lib.ldm_grad_norm(ptrs, sizes, codes, n, 0, 1.0, clip, 64, 64, 1 << 62, None) == ERR_ARG
    # an address and a size whose end passes the largest address
    ends = (ctypes.c_uint64 * 1)((1 << 63) - 64)
    assert lib.ldm_grad_norm(ends, (ctypes.c_int64 * 1)(1 << 20), bytes([code]), 1, 0, 1.0, 1, 64, 64, 1 << 62, None) == ERR_ARG
