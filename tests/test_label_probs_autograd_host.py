"""What autograd can and cannot ask of label_log_probs, without a GPU: the refusal comes before the launch."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from ldmseg import ops


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_derivatives_are_refused(requires_grad):
    """A dual tensor's tangent has no way through the kernels; it must not be dropped without a word."""
    x, t = torch.randn(2, 5, 3), torch.randn(2, 5, 3)
    if requires_grad:
        x.requires_grad_()
    with fw.dual_level():
        d = fw.make_dual(x, t)
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                ops.label_log_probs(d)
        with pytest.raises(RuntimeError, match="GPU tensors only"):          # no dual tensor: only the device is wrong
            ops.label_log_probs(x.detach())
        with pytest.raises(RuntimeError, match="GPU tensors only"):
            ops.label_log_probs(fw.unpack_dual(d).primal.detach())
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda v: ops.label_log_probs(v).entropy, (x.detach(),), (t,))
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        ops.label_log_probs(x)
