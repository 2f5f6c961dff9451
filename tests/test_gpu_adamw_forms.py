"""AdamW and AdamW8bit where the element types of parameters and gradients differ, and where there are more than 2^31 elements."""
import math

import pytest
import torch

from tests.test_gpu_adamw import EPS24, HYPER, _check_step, _cls, _params

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(), (7,), (255,), (256,), (257,), (33, 770), (3, 5, 7), (130, 513), (64, 4096)]


@pytest.mark.parametrize("limit", [None, 0.05])
@pytest.mark.parametrize("p_packed,g_packed", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("p_type,g_type", [(p, g) for p in TYPES for g in TYPES if p != g])
@pytest.mark.parametrize("kind", ["fp32", "8bit"])
def test_gradients_of_another_type(kind, p_type, g_type, p_packed, g_packed, limit):
    """Every step against the definition, each side on vector boundaries or off them."""
    ps = _params(SHAPES, p_type, packed=p_packed)
    for p in ps:
        p.grad_dtype = None      # (lifts the rule that both have one type)
    opt = _cls(kind)(ps, **HYPER, max_grad_norm=limit)
    for k in range(3):
        gs = [g.data for g in _params(SHAPES, g_type, 20 + k, g_packed, 1e-2)]
        for p, g in zip(ps, gs):
            p.grad = g
        norm = math.sqrt(sum((g.double() ** 2).sum().item() for g in gs))
        c = 1.0 if limit is None else min(1.0, limit / (norm + 1e-6))
        _check_step(opt, opt.step, c, 6 * EPS24 if c < 1.0 else 0.0)


def _big(kind, shape, offset):
    """A parameter of more than 2^31 elements with gradients at a few places: the first step moves these by lr, and no other."""
    n = math.prod(shape)
    buf = torch.zeros(n + offset, device="cuda", dtype=torch.bfloat16)
    grad = torch.zeros(n + offset, device="cuda", dtype=torch.bfloat16)
    p = torch.nn.Parameter(buf[offset:].view(shape))
    p.grad = grad[offset:].view(shape)
    spots = [0, 255, 2 ** 31 - 8, 2 ** 31 - 1, 2 ** 31, 2 ** 31 + 12345, n - 300, n - 1]
    for s in spots:
        grad[offset + s] = 0.5
    opt = _cls(kind)([p], lr=0.25, weight_decay=0.0, max_grad_norm=math.inf)
    opt.step()
    assert abs(opt.grad_norm.item() - 0.5 * math.sqrt(len(spots))) < 1e-6
    flat = buf[offset:]
    assert all(flat[s].item() == -0.25 for s in spots)
    assert torch.count_nonzero(flat[: 1 << 31]).item() + torch.count_nonzero(flat[1 << 31:]).item() == len(spots)
    st = opt.state[p]
    for s in spots:      # (1 - b1) g and (1 - b2) g^2, in fp32 or as a code next to it
        if kind == "fp32":
            m, v, tol = st["exp_avg"].view(-1)[s].item(), st["exp_avg_sq"].view(-1)[s].item(), 2 * EPS24
        else:
            at = s // 256
            m = (st["exp_avg_q"].view(-1)[s].float() * st["exp_avg_scale"][at].float()).item()
            v = (st["exp_avg_sq_q"].view(-1)[s].float() * st["exp_avg_sq_scale"][at].float()).item()
            tol = 0.25      # a spacing of e5m2
        assert abs(m / 0.05 - 1.0) <= tol and abs(v / 2.5e-4 - 1.0) <= tol


@pytest.mark.parametrize("kind", ["fp32", "8bit"])
@pytest.mark.parametrize("shape,offset", [((2 ** 31 + 70001,), 0), ((2 ** 31 + 70001,), 1), ((3, 70001, 11, 1000), 0)])
def test_more_than_2_to_the_31_elements(kind, shape, offset):
    """A flat buffer of parameters (one dimension), off the vector boundaries too, and four dimensions."""
    _big(kind, shape, offset)
    torch.cuda.empty_cache()
