"""When GroupNormAct(checkpoint=True) keeps its input: only where a backward can follow.  No GPU: a tensor without memory, the operator's call recorded."""
import pytest
import torch

from elektronn3_amd import norm


class OnGpu(torch.Tensor):
    is_cuda = property(lambda self: True)


@pytest.mark.parametrize('x_grad,w_grad,b_grad,mode,kept', [
    (False, False, False, True, False), (True, False, False, True, True), (False, True, False, True, True), (False, False, True, True, True),
    (True, True, True, False, False), (True, True, True, True, True)])
@pytest.mark.parametrize('affine', [True, False])
def test_kept_where_a_backward_can_follow(monkeypatch, affine, x_grad, w_grad, b_grad, mode, kept):
    seen = []
    monkeypatch.setattr(norm._GroupNormActFunction, 'apply', lambda *a: seen.append(a))
    m = norm.GroupNormAct(2, 8, affine=affine, checkpoint=True)
    if affine:
        m.weight.requires_grad_(w_grad)
        m.bias.requires_grad_(b_grad)
    x = torch.empty(1, 8, 3, 4, 5, device='meta').as_subclass(OnGpu).requires_grad_(x_grad)
    with torch.set_grad_enabled(mode):
        m(x)
    assert seen[0][-1] is (kept and (affine or x_grad))
