"""clip_grad_norm_ against sums in 64 bits: types, sizes, strides, many tensors, values at the ends of the range, refusals."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS24 = 2.0 ** -24
SIZES = [0, 1, 2, 7, 8, 9, 255, 256, 1000, 4097, 70001]


def _grads(sizes, dtypes, scale=1.0, seed=0, offset=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        buf = torch.zeros(n + offset, device="cuda", dtype=dtypes[i % len(dtypes)])
        buf[offset:] = torch.randn(n, device="cuda", generator=gen) * scale
        p = torch.nn.Parameter(torch.zeros_like(buf[offset:]))
        p.grad = buf[offset:]
        out.append(p)
    return out


def _check(ps, limit):
    import came_b200
    old = [p.grad.detach().clone() for p in ps]
    total = sum((g.double() ** 2).sum().item() for g in old)
    want = math.sqrt(total)
    norm = came_b200.clip_grad_norm_(ps, limit)
    assert norm.shape == () and norm.dtype == torch.float32 and norm.device == ps[0].device
    # eight squares in fp32 (nine half steps at most, halved by the root), and the rounding of the result
    assert abs(norm.item() - want) <= 6 * EPS24 * want
    c = min(1.0, limit / (want + 1e-6))
    for p, g in zip(ps, old):
        f = torch.finfo(g.dtype)
        if c == 1.0:
            assert torch.equal(p.grad, g)
            continue
        x = g.double() * c
        tiny = f.smallest_normal * f.eps / 2
        assert ((p.grad.double() - x).abs() <= (f.eps / 2 * 1.01 + 8 * EPS24) * x.abs() + tiny).all()


@pytest.mark.parametrize("offset", [0, 1, 3])
@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float16,), (torch.float32, torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("limit", [1.0, 1e6, math.inf, 0.0])
def test_norm_and_scaling(dtypes, limit, offset):
    _check(_grads(SIZES, dtypes, offset=offset), limit)


@pytest.mark.parametrize("count", [1, 64, 65, 1024, 1025, 2500])
def test_many_tensors(count):
    _check(_grads([3 + (17 * i) % 50 for i in range(count)], (torch.bfloat16, torch.float32)), 0.5)


@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e18, 1e30])
def test_range(scale):
    """Squares outside the range of fp32."""
    import came_b200
    ps = _grads([5000, 3], (torch.float32,), scale)
    want = math.sqrt(sum((p.grad.double() ** 2).sum().item() for p in ps))
    assert abs(came_b200.clip_grad_norm_(ps, math.inf).item() - want) <= 6 * EPS24 * want
    _check(ps, want / 4 if scale > 1 else 1.0)


def test_zero_and_nothing():
    import came_b200
    ps = _grads([100, 0], (torch.float32,), 0.0)
    assert came_b200.clip_grad_norm_(ps, 1.0).item() == 0.0 and not ps[0].grad.any()
    empty = _grads([0], (torch.float32,))
    assert came_b200.clip_grad_norm_(empty, 1.0).item() == 0.0
    assert came_b200.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3, device="cuda"))], 1.0).item() == 0.0
    assert came_b200.clip_grad_norm_([], 1.0).item() == 0.0
    assert came_b200.clip_grad_norm_(ps[0], 1.0).item() == 0.0
    assert came_b200.clip_grad_norm_((p for p in ps), 1.0).item() == 0.0


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_not_finite(bad):
    """As torch's: with an infinite norm the factor is zero, with one that is not a number everything becomes it."""
    import came_b200
    ps = _grads([300, 20], (torch.float32,))
    ps[1].grad[4] = bad
    keep = [p.grad.clone() for p in ps]
    with pytest.raises(RuntimeError, match="norm"):
        came_b200.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
    assert torch.equal(ps[0].grad, keep[0])
    assert came_b200.clip_grad_norm_(ps, math.inf).item() != 1.0 and torch.equal(ps[0].grad, keep[0])
    norm = came_b200.clip_grad_norm_(ps, 1.0).item()
    if math.isnan(bad):
        assert math.isnan(norm) and torch.isnan(ps[0].grad).all()
    else:
        assert norm == math.inf and not ps[0].grad.any() and math.isnan(ps[1].grad[4].item())


def test_strides():
    wide = torch.randn(50, 60, device="cuda")
    keep = wide.clone()
    ps = [torch.nn.Parameter(torch.zeros(50, 20, device="cuda")), torch.nn.Parameter(torch.zeros(30, 40, device="cuda"))]
    ps[0].grad = wide[:, 10:30]
    ps[1].grad = torch.randn(40, 30, device="cuda").t()
    _check(ps, 1.0)
    assert torch.equal(wide[:, :10], keep[:, :10]) and torch.equal(wide[:, 30:], keep[:, 30:]) and not torch.equal(wide, keep)
    ps[0].grad = torch.ones(20, device="cuda").expand(50, 20)
    import came_b200
    assert abs(came_b200.clip_grad_norm_(ps[:1], math.inf).item() - math.sqrt(1000.0)) < 1e-4
    with pytest.raises(RuntimeError):
        came_b200.clip_grad_norm_(ps[:1], 1.0)


def test_side_stream_and_capture():
    import came_b200
    ps = _grads([1000, 77, 20000], (torch.bfloat16,))
    want = math.sqrt(sum((p.grad.double() ** 2).sum().item() for p in ps))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        norm = came_b200.clip_grad_norm_(ps, math.inf)
    side.synchronize()
    assert abs(norm.item() - want) <= 6 * EPS24 * want
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = came_b200.clip_grad_norm_(ps, 1.0)
    for k in (1.0, 3.0):
        for i, p in enumerate(ps):
            p.grad.copy_(_grads([p.numel()], (torch.bfloat16,), k, i)[0].grad)
        want = math.sqrt(sum((p.grad.double() ** 2).sum().item() for p in ps))
        graph.replay()
        torch.cuda.synchronize()
        assert abs(norm.item() - want) <= 6 * EPS24 * want
        after = math.sqrt(sum((p.grad.double() ** 2).sum().item() for p in ps))
        assert abs(after - 1.0) <= 2.0 ** -8
    a, b = came_b200.clip_grad_norm_(ps, 1.0), came_b200.clip_grad_norm_(ps, 0.5)      # two calls: two results
    assert a.item() > 0.9 and a.data_ptr() != b.data_ptr()


def test_refusals():
    import came_b200
    ps = _grads([10, 20], (torch.float32,))
    with pytest.raises(ValueError, match="twice"):
        came_b200.clip_grad_norm_([ps[0], ps[0]], 1.0)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            came_b200.clip_grad_norm_(ps, bad)
    with pytest.raises(ValueError):
        came_b200.clip_grad_norm_(ps, 1.0, norm_type=math.inf)
    ps[1].grad = None
    d = torch.nn.Parameter(torch.zeros(3, device="cuda", dtype=torch.float64))
    d.grad = torch.ones_like(d)
    with pytest.raises(RuntimeError, match="float64"):
        came_b200.clip_grad_norm_([ps[0], d], 1.0)
    c = torch.nn.Parameter(torch.zeros(3))
    c.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="CPU"):
        came_b200.clip_grad_norm_([ps[0], c], 1.0)
    s = torch.nn.Parameter(torch.zeros(4, 4, device="cuda"))
    s.grad = torch.sparse_coo_tensor(torch.tensor([[0], [0]]), torch.tensor([1.0]), (4, 4)).cuda()
    with pytest.raises(RuntimeError, match="sparse"):
        came_b200.clip_grad_norm_([s], 1.0)
