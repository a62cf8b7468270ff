"""What a refused clip leaves behind: gradients, and what autograd knows of them, as they were."""
import pytest
import torch

from ldmseg.ops import native as K
from ldmseg.trainers import clip_grad_norm_

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _param(n, dtype=torch.float32, device=DEV):
    p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device=device))
    p.grad = torch.full((n,), 3.0, dtype=dtype, device=device)
    return p


def test_a_refused_clip_marks_nothing_as_modified():
    """A graph that has saved a gradient can still run backward after a clip that was refused: nothing was written."""
    def overlap(p):
        q = torch.nn.Parameter(torch.zeros(2, device=DEV))
        q.grad = p.grad[1:3]
        return [p, q]

    def dense(p):
        q = _param(4)
        q.grad = torch.ones(1, device=DEV).expand(4)
        return [p, q]

    refused = [
        (ValueError, lambda p: [p, _param(4, device="cpu")], {}), (ValueError, overlap, {}), (ValueError, dense, {}),
        (TypeError, lambda p: [p, _param(4, torch.float16)], {}), (TypeError, lambda p: [p, 7], {}),
        (ValueError, lambda p: [p], {"max_norm": -1.0}), (ValueError, lambda p: [p], {"norm_type": 3.0}),
    ]
    for exc, params, kw in refused:
        p = _param(4)
        w = torch.ones(4, device=DEV, requires_grad=True)
        y = (w * p.grad).sum()
        version = p.grad._version
        with pytest.raises(exc):
            clip_grad_norm_(params(p), **{"max_norm": 1.0, **kw})
        assert p.grad._version == version and (p.grad == 3).all()
        y.backward()
        assert (w.grad == 3).all()
    a = torch.full((5,), 2.0, device=DEV)
    version = a._version
    with torch.inference_mode():
        q = torch.ones(3, device=DEV)
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        K.clip_grads([a, q], 1.0)
    assert a._version == version and (a == 2).all() and (q == 1).all()


def test_a_clip_marks_every_gradient_as_modified_once():
    ps = [_param(4), _param(100_000, torch.bfloat16), _param(0)]
    versions = [p.grad._version for p in ps]
    clip_grad_norm_(ps, 1.0)
    assert [p.grad._version for p in ps] == [v + 1 for v in versions]
    K.grad_norm([p.grad for p in ps])
    assert [p.grad._version for p in ps] == [v + 1 for v in versions]
    with torch.inference_mode():                                # there it may be written, as any tensor
        q = torch.full((3,), 4.0, device=DEV)
        assert K.clip_grads([q], 1.0) > 6 and (q < 1).all()
