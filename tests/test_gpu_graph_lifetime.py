"""Captured steps beside eager ones whose tensors lie elsewhere: what a graph reads stays, and a schedule reaches it."""
import copy
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = [(64, 96), (300,), (33, 70)]


def _params(dtype=torch.bfloat16, seed=3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(s, device="cuda", generator=gen) * 0.05).to(dtype)) for s in SHAPES]


def _grads(ps, seed, offset=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for p in ps:
        buf = torch.zeros(p.numel() + offset, device="cuda", dtype=p.dtype)
        buf[offset:] = torch.randn(p.numel(), device="cuda", generator=gen) * 1e-2
        out.append(buf[offset:].view(p.shape))
    return out


def _make(name, ps, **kw):
    import came_b200
    return getattr(came_b200, name)(ps, lr=1e-3, weight_decay=1e-2, **kw)


def _capture(opt):
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    return graph


def _same(ps, a, qs, b):
    for p, q in zip(ps, qs):
        assert torch.equal(p.data, q.data)
        for key, v in a.state[p].items():
            if torch.is_tensor(v):
                w = b.state[q][key]
                assert torch.equal(v.view(torch.uint8) if "float8" in str(v.dtype) else v, w.view(torch.uint8) if "float8" in str(w.dtype) else w), key


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("name", ["AdamW", "AdamW8bit", "CAME8bit", "CAMECUDA"])
def test_replays_between_eager_steps_with_moved_gradients(name, offset):
    """offset 1: the moved gradients start on no boundary, which asks for another plan in any case.  (The order in which the CAME
    kernels add goes by the alignment: the twin's gradients lie as those of the step they stand for.)"""
    ps, qs = _params(), _params()
    graphed, eager = _make(name, ps), _make(name, qs)
    own = _grads(ps, 1)
    for p, g in zip(ps, own):
        p.grad = g
    graphed.prime_for_cuda_graph()
    graph = _capture(graphed)
    for k in range(6):
        gs = _grads(ps, 10 + k, offset if k % 2 else 0)
        for group in (*graphed.param_groups, *eager.param_groups):
            group["lr"] = 1e-3 * 0.5 ** k
        for q, g in zip(qs, gs):
            q.grad = g
        eager.step()
        if k % 2:      # an eager step, and what it may leave unused
            for p, g in zip(ps, gs):
                p.grad = g
            graphed.step()
            torch.cuda.synchronize()
            del gs
        else:
            for h, g in zip(own, gs):
                h.copy_(g)
            graphed.update_captured_hypers()
            graph.replay()
            torch.cuda.synchronize()
    _same(ps, graphed, qs, eager)


@pytest.mark.parametrize("name", ["AdamW8bit", "CAME8bit"])
def test_a_loaded_state_is_not_the_graphs(name):
    """load_state_dict makes new state tensors: a graph from before goes on with those it was captured with."""
    ps = _params()
    opt = _make(name, ps)
    for p, g in zip(ps, _grads(ps, 1)):
        p.grad = g
    opt.prime_for_cuda_graph()
    graph = _capture(opt)
    graph.replay()
    opt.load_state_dict(copy.deepcopy(opt.state_dict()))
    want = copy.deepcopy(opt.state_dict()["state"])
    before = [p.detach().clone() for p in ps]
    graph.replay()
    torch.cuda.synchronize()
    assert all(not torch.equal(b, p.data) for b, p in zip(before, ps))
    for key, st in opt.state_dict()["state"].items():
        for k, v in st.items():
            if torch.is_tensor(v):
                assert torch.equal(v.float(), want[key][k].float())


def test_addresses_of_a_captured_plan_stay():
    from came_b200 import _lib
    ps = _params()
    opt = _make("AdamW", ps)
    for p, g in zip(ps, _grads(ps, 1)):
        p.grad = g
    opt.prime_for_cuda_graph()
    (plan,) = opt._engine.plans.values()
    assert plan.captured == 0
    graph = _capture(opt)
    assert plan.captured == 1
    lib, n = _lib.load(), len(ps)
    stream = torch.cuda.current_stream().cuda_stream
    same = (C.c_void_p * n)(*[p.grad.data_ptr() for p in ps])
    keep = _grads(ps, 2)
    other = (C.c_void_p * n)(*[g.data_ptr() for g in keep])
    assert lib.came_b200_plan_set_pointers(plan.handle, same, None, n, stream) == _lib.OK
    assert lib.came_b200_plan_set_pointers(plan.handle, other, None, n, stream) == _lib.E_INVALID
    assert b"captured" in lib.came_b200_last_error()
    graph.replay()
    torch.cuda.synchronize()


def test_a_capture_that_would_need_a_new_plan_is_refused():
    ps = _params()
    opt = _make("AdamW", ps)
    for p, g in zip(ps, _grads(ps, 1)):
        p.grad = g
    opt.prime_for_cuda_graph()
    first = _capture(opt)
    for p, g in zip(ps, _grads(ps, 2)):
        p.grad = g
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="prime_for_cuda_graph"):
        _capture(opt)
    opt.prime_for_cuda_graph()      # as the message says
    second = _capture(opt)
    first.replay()
    second.replay()
    torch.cuda.synchronize()
    assert opt.state[ps[0]]["step"].item() == 2


@pytest.mark.parametrize("name", ["AdamW", "AdamW8bit"])
@pytest.mark.parametrize("limit", [None, 0.01])
def test_the_clip_is_switched_around_a_capture(name, limit):
    """The graph goes on as it was captured, eager steps follow the switch, and a schedule for the graph is refused."""
    ps, qs = _params(), _params()
    opt, twin = _make(name, ps, max_grad_norm=limit), _make(name, qs, max_grad_norm=limit)
    gs = _grads(ps, 1)
    for p, q, g in zip(ps, qs, gs):
        p.grad = q.grad = g
    opt.prime_for_cuda_graph()
    graph = _capture(opt)
    graph.replay()
    twin.step()
    for o in (opt, twin):
        o.max_grad_norm = None if limit else 0.01
    with pytest.raises(ValueError, match="captured"):
        opt.update_captured_hypers()
    opt.step(), twin.step()
    with pytest.raises(ValueError, match="captured"):
        opt.update_captured_hypers()
    graph.replay()
    twin.max_grad_norm = limit
    twin.step()
    torch.cuda.synchronize()
    _same(ps, opt, qs, twin)
    opt.prime_for_cuda_graph()
    graph = _capture(opt)      # a capture of the new setting: it may be updated
    opt.update_captured_hypers()
    graph.replay()
    twin.max_grad_norm = opt.max_grad_norm
    twin.step()
    torch.cuda.synchronize()
    _same(ps, opt, qs, twin)


@pytest.mark.parametrize("name", ["AdamW", "AdamW8bit"])
def test_empty_parameters_step_by_the_table(name):
    import came_b200
    ps, qs = _params(), _params()
    empty = [torch.nn.Parameter(torch.zeros(s, device="cuda", dtype=torch.bfloat16)) for s in ((0,), (4, 0))]
    opt, twin = getattr(came_b200, name)([empty[0], *ps, empty[1]], lr=1e-3), getattr(came_b200, name)(qs, lr=1e-3)
    for k in range(4):
        for p, q, g in zip(ps, qs, _grads(ps, 5 + k)):
            p.grad = q.grad = g
        for e in empty:
            e.grad = torch.zeros_like(e) if k != 2 else None
        opt.step(), twin.step()
        assert opt._table is not None
    torch.cuda.synchronize()
    _same(ps, opt, qs, twin)


@pytest.mark.parametrize("name", ["AdamW", "AdamW8bit"])
def test_the_norm_belongs_to_its_plan(name):
    ps = _params()
    opt = _make(name, ps, max_grad_norm=1.0)
    own = _grads(ps, 1)
    for p, g in zip(ps, own):
        p.grad = g
    opt.prime_for_cuda_graph()
    assert opt.grad_norm is None
    graph = _capture(opt)
    captured = opt.grad_norm
    for p, g in zip(ps, _grads(ps, 2)):
        p.grad = g * 3
    opt.step()
    graph.replay()
    torch.cuda.synchronize()
    for norm, gs in ((captured, own), (opt.grad_norm, [p.grad for p in ps])):
        want = sum((g.double() ** 2).sum().item() for g in gs) ** 0.5
        assert abs(norm.item() - want) <= 6 * 2.0 ** -24 * want


@pytest.mark.parametrize("name", ["AdamW8bit", "CAME8bit"])
def test_an_eager_step_between_a_capture_with_other_gradients_and_its_first_replay(name):
    """The capture moves the plan to other gradients, but its upload of their addresses has not run yet."""
    ps, qs = _params(), _params()
    opt, twin = _make(name, ps), _make(name, qs)
    first, gs = _grads(ps, 1), _grads(ps, 2)
    for p, g in zip(ps, first):
        p.grad = g
    opt.prime_for_cuda_graph()
    for p, q, g in zip(ps, qs, gs):
        p.grad = q.grad = g
    graphs = [_capture(opt), _capture(opt)]      # (the second finds the plan moved)
    opt.step(), twin.step()
    torch.cuda.synchronize()
    _same(ps, opt, qs, twin)
    for graph in graphs:
        graph.replay()
        twin.step()
    torch.cuda.synchronize()
    _same(ps, opt, qs, twin)


@pytest.mark.parametrize("name", ["AdamW8bit", "CAME8bit"])
def test_two_captures_with_other_gradients_before_any_step(name):
    ps, qs = _params(), _params()
    opt, twin = _make(name, ps), _make(name, qs)
    first, gs = _grads(ps, 1), _grads(ps, 2)
    for p, g in zip(ps, first):
        p.grad = g
    opt.prime_for_cuda_graph()
    for p, q, g in zip(ps, qs, gs):
        p.grad = q.grad = g
    _, second = _capture(opt), _capture(opt)
    second.replay()      # the first never runs
    twin.step()
    torch.cuda.synchronize()
    _same(ps, opt, qs, twin)


@pytest.mark.parametrize("name", ["AdamW8bit", "CAME8bitFull"])
def test_a_copy_goes_on_like_the_original(name):
    opt = _make(name, _params())
    ps = opt.param_groups[0]["params"]
    for p, g in zip(ps, _grads(ps, 1)):
        p.grad = g
    opt.step()
    other = copy.deepcopy(opt)
    qs = other.param_groups[0]["params"]
    for p, q, g in zip(ps, qs, _grads(ps, 2)):
        p.grad = q.grad = g
    opt.step(), other.step()
    torch.cuda.synchronize()
    assert all(p is not q for p, q in zip(ps, qs))
    _same(ps, opt, qs, other)
