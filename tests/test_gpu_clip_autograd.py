"""What clip_grad_norm_ is to autograd: an operation in place on the gradients, and a reading one where the norm alone is asked for."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _param(n, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.nn.Parameter(torch.randn(n, device="cuda", generator=gen))


def test_versions_count_what_is_scaled():
    import came_b200
    ps = [_param(100), _param(7, 1), _param(64, 2)]
    ps[0].grad, ps[1].grad = torch.ones(100, device="cuda"), torch.ones(7, device="cuda")
    wide = torch.ones(8, 20, device="cuda")
    ps.append(torch.nn.Parameter(torch.zeros(8, 10, device="cuda")))
    ps[3].grad = wide[:, :10]      # (copied, scaled and copied back)
    for which in (ps[:3], ps):
        before = [p.grad._version for p in which if p.grad is not None]
        came_b200.clip_grad_norm_(which, math.inf)
        assert [p.grad._version for p in which if p.grad is not None] == before
        came_b200.clip_grad_norm_(which, 0.5)
        assert all(p.grad._version > b for p, b in zip([p for p in which if p.grad is not None], before))


def test_a_double_backward_through_a_clipped_gradient_is_refused():
    import came_b200
    p = _param(50)
    (g,) = torch.autograd.grad((p ** 3).sum(), p, create_graph=True)
    z = (g * g).sum()      # keeps g
    p.grad = g
    came_b200.clip_grad_norm_([p], math.inf)
    (want,) = torch.autograd.grad(z, p, retain_graph=True)
    assert torch.allclose(want, 36 * p.detach() ** 3)
    came_b200.clip_grad_norm_([p], 0.1)
    with pytest.raises(RuntimeError, match="inplace operation"):
        torch.autograd.grad(z, p)


def test_a_lazy_copy_keeps_the_unclipped_gradient():
    import came_b200
    p = _param(300)
    keep = torch.randn(300, device="cuda")
    want = keep.clone()
    p.grad = torch._lazy_clone(keep)
    came_b200.clip_grad_norm_([p], 0.1)
    assert torch.equal(keep, want) and abs(p.grad.norm().item() - 0.1) < 1e-4
