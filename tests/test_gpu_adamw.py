"""AdamW and AdamW8bit against the definition in 64 bits, one step at a time from the kernel's own state before it; what a
step must leave alone; captured, moved, sharded and resumed steps."""
import copy
import math
import warnings

import pytest
import torch

from tests import adamw_ref as ref

pytestmark = pytest.mark.gpu

EPS24 = 2.0 ** -24
SHAPES = [(), (1,), (7,), (0,), (8,), (255,), (256,), (257,), (33, 770), (3, 5, 7), (6, 2, 3, 3), (4096,), (130, 513), (64, 4096)]
HYPER = dict(lr=2e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def _cls(kind):
    import came_b200
    return {"fp32": came_b200.AdamW, "8bit": came_b200.AdamW8bit}[kind]


def _params(shapes, dtype, seed=0, packed=False, scale=0.05):
    """Parameters of their own, or one behind the other in one buffer from its second element on (no 16-byte boundaries)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    total = sum(math.prod(s) for s in shapes)
    buf = torch.zeros(total + 1, device="cuda", dtype=dtype)
    out, at = [], 1
    for s in shapes:
        x = (torch.randn(s, device="cuda", generator=gen) * scale).to(dtype)
        if packed:
            v = buf[at: at + x.numel()].view(s)
            v.copy_(x)
            at += x.numel()
            x = v
        out.append(torch.nn.Parameter(x))
    return out


def _set_grads(ps, seed, scale=1e-2, packed=False):
    gs = _params([tuple(p.shape) for p in ps], ps[0].dtype, seed, packed, scale)
    for p, g in zip(ps, gs):
        p.grad = g.data
    return gs


def _state(opt, p):
    """(m, v, t) of a parameter in 64 bits; zeros before the first step."""
    st = opt.state[p] if p in opt.state else {}
    if "step" not in st:
        z = torch.zeros(p.shape, dtype=torch.float64, device=p.device)
        return z, z.clone(), 0
    t = int(st["step"].item())
    if "exp_avg" in st:
        return st["exp_avg"].double(), st["exp_avg_sq"].double(), t
    return ref.decode(st["exp_avg_q"], st["exp_avg_scale"]).double(), ref.decode(st["exp_avg_sq_q"], st["exp_avg_sq_scale"]).double(), t


def _check_step(opt, step, c=1.0, c_err=0.0, hyper=None):
    """Takes `step()` and holds every parameter and state to the definition.  c: factor of the gradients, c_err its relative error."""
    before = []
    for gi, group in enumerate(opt.param_groups):
        for p in group["params"]:
            if p.grad is not None and p.numel():
                before.append((group, p, p.detach().clone(), p.grad.detach().clone(), *_state(opt, p)))
    step()
    torch.cuda.synchronize()
    for group, p, old, g, m, v, t in before:
        h = {k: group[k] for k in ("lr", "betas", "eps")}
        g64 = g.double() * (c * group.get("grad_scale", 1.0))
        m64, v64, m_mag, v_mag = ref.moments(m, v, g64, h["betas"])
        st = opt.state[p]
        assert int(st["step"].item()) == t + 1
        # c and its rounding, the constants' roundings, products and sum: 5 half steps for m, 8 for v (g twice)
        m_tol = (5 * EPS24 + c_err) * m_mag + 1e-44
        v_tol = (8 * EPS24 + 2 * c_err) * v_mag + 1e-44
        if "exp_avg" in st:
            assert ((st["exp_avg"].double() - m64).abs() <= m_tol).all()
            assert ((st["exp_avg_sq"].double() - v64).abs() <= v_tol).all()
        else:
            _check_codes(st["exp_avg_q"], st["exp_avg_scale"], m64, m_tol, "m", t + 1)
            _check_codes(st["exp_avg_sq_q"], st["exp_avg_sq_scale"], v64, v_tol, "v", t + 1)
        p64, upd = ref.param(old.double(), m64, v64, t + 1, wd=group["weight_decay"], **h)
        # (a moment that is almost nothing of its two terms: its own bound instead of one relative to it)
        slack = h["lr"] / (1 - h["betas"][0] ** (t + 1)) * m_tol / (v64.sqrt() / (1 - h["betas"][1] ** (t + 1)) ** 0.5 + h["eps"])
        slack = slack + upd.abs() * 1e-44 / v64.clamp(min=1e-60)      # (a v next to nothing: its last bit is more than a rounding)
        err, tol = (p.detach().double() - p64).abs(), ref.param_bound(p64, upd, p.dtype) + (1.02 + 4 * c_err) * slack + c_err * upd.abs()
        tol = torch.where(torch.isfinite(tol), tol, torch.zeros_like(tol))
        assert (err <= tol).all(), (tuple(p.shape), (err - tol).max().item())


def _check_codes(codes, scale, x64, tol, which, t):
    """Codes within a spacing of the value; equal to the rounding of the 64-bit value wherever its error cannot reach the border."""
    n = x64.numel()
    top, drop, least, _, kept, _ = ref.FORMATS[which]
    big = ref.blocks(x64.abs()).amax(1)
    s = scale.double()[: big.numel()]
    ok = (s == torch.exp2(torch.floor(torch.log2(big.clamp(min=1e-300))) - top).clamp(min=2.0 ** -126))
    edge = torch.exp2(torch.round(torch.log2(big.clamp(min=1e-300))))      # next to a power of two either exponent will do
    near = (big - edge).abs() <= 16 * EPS24 * edge
    assert (ok | near).all()
    sc = s.repeat_interleave(256)[:n].view(x64.shape)
    y, got = x64 / sc, codes.float().double()
    if least is not None:
        whole = (ref.blocks(x64).amax(1) > 0).repeat_interleave(256)[:n].view(x64.shape)
        y = torch.where(whole, y.clamp(min=least), y)
    step = ref.spacing(y, which).double()
    ytol = tol / sc
    assert ((got - y).abs() <= step * (1 + 2.0 ** -6) + ytol).all()
    # the rounding itself: floor(|y| / u + r / 2^drop) * u, u the spacing before the format's subnormals
    h = ref.random_bits(n, t, x64.device).view(x64.shape)
    r = ((h & 0xFFFFF) if which == "m" else h >> 11).double() / 2.0 ** drop
    u = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -120))) - kept)
    q = y.abs() / u + r
    sure = (q - torch.round(q)).abs() > ytol / u + 2.0 ** -19      # (r is whole units of 2^-drop: a border lies on the grid of q)
    sure &= y.abs() > 2.0 ** -5 if which == "m" else y.abs() > 2.0 ** -13
    want = torch.floor(q) * u * torch.sign(y)
    assert (got[sure] == want[sure]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("kind", ["fp32", "8bit"])
def test_steps_follow_the_definition(kind, dtype, packed):
    ps = _params(SHAPES, dtype, packed=packed)
    opt = _cls(kind)(ps, **HYPER)
    for k in range(4):
        gs = _set_grads(ps, 100 + k, 1e-2 * 10.0 ** -k, packed)
        if k == 2:
            ps[5].grad = None      # a parameter that misses a step: its own count
        _check_step(opt, opt.step)
        assert all(torch.equal(p.grad, g) for p, g in zip(ps, gs) if p.grad is not None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("packed", [False, True])
def test_codes_equal_those_of_separate_fp32_operations(dtype, packed):
    """Moments formed by one tensor operation per product and sum, rounded by the oracle: the same bytes, at any scale."""
    ps = _params([(70000,), (129, 1026), (257,), (64, 4096), (9000,)], dtype, packed=packed)
    opt = _cls("8bit")(ps, lr=1e-3, betas=(0.9, 0.99))
    opt.param_groups[0]["grad_scale"] = 0.125
    for k, scale in enumerate((1e-2, 1e-2, 1e-5, 1e-3, 1.0)):
        _set_grads(ps, k, scale, packed)
        if dtype == torch.float32 and k == 3:      # blocks next to underflow, some of them zero
            ps[0].grad *= 10.0 ** -torch.arange(0, 40, 4, device="cuda").repeat_interleave(7000)
            ps[2].grad[:] = 0.0
        before = {p: _state(opt, p) for p in ps}
        opt.step()
        for p in ps:
            m, v, t = before[p]
            g = p.grad.float() * 0.125
            m, v = m.float() * 0.9 + g * (1.0 - 0.9), v.float() * 0.99 + g * g * (1.0 - 0.99)
            st = opt.state[p]
            for x, which, key in ((m, "m", "exp_avg"), (v, "v", "exp_avg_sq")):
                codes, scales = ref.encode(x, which, t + 1)
                assert torch.equal(scales, st[key + "_scale"].float())
                assert torch.equal(codes.view(torch.uint8), st[key + "_q"].view(torch.uint8)), (tuple(p.shape), which, k)


@pytest.mark.parametrize("hyper", [dict(betas=(0.0, 0.0)), dict(betas=(0.0, 0.95)), dict(betas=(0.95, 0.5), eps=1.0), dict(lr=0.0),
                                   dict(weight_decay=0.0), dict(betas=(0.9, 0.99999), lr=1.0), dict(eps=1e-20, weight_decay=0.5)])
@pytest.mark.parametrize("kind", ["fp32", "8bit"])
def test_hyper_parameters(kind, hyper):
    ps = _params([(257,), (40, 64), (300, 7)], torch.float32)
    opt = _cls(kind)([{"params": ps[:1], "lr": 0.5}, {"params": ps[1:]}], **{**HYPER, **hyper})
    for k in range(3):
        _set_grads(ps, k)
        _check_step(opt, opt.step)
        opt.param_groups[0]["lr"] *= 0.5
        opt.param_groups[1]["betas"] = (0.8, 0.9)


@pytest.mark.parametrize("kind", ["fp32", "8bit"])
@pytest.mark.parametrize("scale", [0.0, 1e-25, 1e-12, 1e12])
def test_gradient_ranges(kind, scale):
    ps = _params([(1000,), (64, 96)], torch.float32)
    opt = _cls(kind)(ps, **HYPER)
    for k in range(3):
        _set_grads(ps, k, scale)
        if k == 1:
            ps[0].grad[:300] = 0.0
        _check_step(opt, opt.step)
    if scale == 0.0:
        st = opt.state[ps[0]]
        assert not any(v.float().any() for key, v in st.items() if key in ("exp_avg", "exp_avg_sq", "exp_avg_q", "exp_avg_sq_q"))


@pytest.mark.parametrize("kind", ["fp32", "8bit"])
@pytest.mark.parametrize("eps", [1e-20, 1e-15, 1e-11, 1e-9])
def test_second_moments_next_to_nothing(kind, eps):
    """Roots of numbers at the lower end of fp32 beside an eps of their size."""
    ps = _params([(1000,), (64, 96)], torch.float32)
    opt = _cls(kind)(ps, **{**HYPER, "eps": eps, "betas": (0.9, 0.9999)})
    for k in range(3):
        _set_grads(ps, k, 3e-17)
        ps[1].grad *= 10.0 ** torch.arange(-2, 4, device="cuda").repeat(16)
        _check_step(opt, opt.step)


def test_agrees_with_torch_and_loads_its_checkpoint():
    ps, qs = _params(SHAPES, torch.float32), _params(SHAPES, torch.float32)
    ours, theirs = _cls("fp32")(ps, **HYPER), torch.optim.AdamW(qs, **HYPER)
    for k in range(6):
        if k == 3:      # go on from torch's state, in a new optimizer
            ours = _cls("fp32")(ps, **HYPER)
            ours.load_state_dict(copy.deepcopy(theirs.state_dict()))
            for p, q in zip(ps, qs):
                p.data.copy_(q.data)
        _set_grads(ps, k)
        for p, q in zip(ps, qs):
            q.grad = p.grad.clone()
        ours.step()
        theirs.step()
        for p, q in zip(ps, qs):
            # six steps of an update of lr, each with some ten fp32 roundings on either side
            assert torch.allclose(p.data, q.data, rtol=12 * EPS24, atol=6 * 40 * EPS24 * HYPER["lr"])
            if p.numel():
                assert ours.state[p]["step"].item() == k + 1
    with pytest.raises(ValueError, match="amsgrad"):
        ours.load_state_dict(torch.optim.AdamW(qs, amsgrad=True).state_dict())


@pytest.mark.parametrize("kind", ["fp32", "8bit"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_state_dict_round_trip(kind, dtype):
    ps, qs = _params(SHAPES, dtype), _params(SHAPES, dtype)
    a, b = _cls(kind)(ps, **HYPER), _cls(kind)(qs, **HYPER)
    for k in range(2):
        _set_grads(ps, k)
        a.step()
    b.load_state_dict(copy.deepcopy(a.state_dict()))
    for p, q in zip(ps, qs):
        q.data.copy_(p.data)
    _set_grads(ps, 7), _set_grads(qs, 7)
    a.step(), b.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p.data, q.data)
        for key, v in a.state[p].items():
            w = b.state[q][key]
            assert w.dtype == v.dtype and torch.equal(v.view(torch.uint8) if "float8" in str(v.dtype) else v,
                                                      w.view(torch.uint8) if "float8" in str(w.dtype) else w), key
    other = _cls("8bit" if kind == "fp32" else "fp32")(qs, **HYPER)
    other.load_state_dict(copy.deepcopy(a.state_dict()))
    with pytest.raises(RuntimeError, match="another optimizer"):
        other.step()


@pytest.mark.parametrize("kind", ["fp32", "8bit"])
def test_strides(kind):
    """Parameters and gradients that are not contiguous, and elements between them that must stay."""
    wide = torch.randn(70, 80, device="cuda")
    keep = wide.clone()
    ps = [torch.nn.Parameter(wide[:, 3:40]), torch.nn.Parameter(torch.randn(96, 33, device="cuda").t()),
          torch.nn.Parameter(torch.randn(4, 8, 5, 5, device="cuda").to(memory_format=torch.channels_last))]
    opt = _cls(kind)(ps, **HYPER)
    for k in range(2):
        for p in ps:
            p.grad = torch.randn(p.shape, device="cuda") if k else torch.randn(p.shape[::-1], device="cuda").permute(*reversed(range(p.dim())))
        _check_step(opt, opt.step)
    assert torch.equal(wide[:, :3], keep[:, :3]) and torch.equal(wide[:, 40:], keep[:, 40:])


@pytest.mark.parametrize("offset", [0, 4, 8])
@pytest.mark.parametrize("kind", ["fp32", "8bit"])
def test_nothing_beyond_the_tensor_is_written(kind, offset):
    """Sentinels on both sides of parameters and states, states off their boundaries."""
    n = 3000 + 13
    buf = torch.full((n + 64,), 5.0, device="cuda", dtype=torch.bfloat16)
    p = torch.nn.Parameter(buf[32: 32 + n])
    p.grad = torch.ones_like(p)
    opt = _cls(kind)([p], **HYPER)
    opt.prime_for_cuda_graph()
    st, around = opt.state[p], []
    for key in [k for k in st if k != "step"]:
        raw = torch.full((st[key].numel() * st[key].element_size() + 1024,), 77, device="cuda", dtype=torch.uint8)
        at = 512 + (offset if st[key].element_size() == 4 else offset // 4 * 3)
        mid = raw[at: at + st[key].numel() * st[key].element_size()]
        mid.copy_(st[key].view(torch.uint8).reshape(-1))
        st[key] = mid.view(st[key].dtype).view(st[key].shape)
        around.append((raw, at, mid.numel()))
    opt.prime_for_cuda_graph()
    _check_step(opt, opt.step)
    assert (buf[:32] == 5.0).all() and (buf[32 + n:] == 5.0).all()
    assert all(v.float().ne(0).all() for key, v in st.items() if key in ("exp_avg", "exp_avg_sq", "exp_avg_q", "exp_avg_sq_q"))
    for raw, at, k in around:
        assert (raw[:at] == 77).all() and (raw[at + k:] == 77).all()


@pytest.mark.parametrize("kind", ["fp32", "8bit"])
@pytest.mark.parametrize("limit", [1e-3, 1e3, math.inf])
def test_clip_inside_the_step(kind, limit):
    ps = _params(SHAPES, torch.float32)
    opt = _cls(kind)([{"params": ps[:9], "grad_scale": 0.5}, {"params": ps[9:], "weight_decay": 0.0}], **HYPER, max_grad_norm=limit)
    assert opt.grad_norm is None
    for k in range(2):
        gs = _set_grads(ps, k)
        total = sum(((g.double() * (0.5 if i < 9 else 1.0)) ** 2).sum().item() for i, g in enumerate(gs))
        c = min(1.0, limit / (math.sqrt(total) + 1e-6))
        # eight squares in fp32: nine half steps of the sum at most, half of that in its root; the factor's own rounding
        _check_step(opt, opt.step, c, 6 * EPS24 if c < 1 else 0.0)
        assert abs(opt.grad_norm.item() - math.sqrt(total)) <= 6 * EPS24 * math.sqrt(total)
    before = [p.detach().clone() for p in ps]
    opt.max_grad_norm = None      # (another plan)
    _check_step(opt, opt.step)
    assert opt.grad_norm is None and not torch.equal(before[-1], ps[-1].data)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("kind", ["fp32", "8bit"])
def test_a_norm_that_is_not_finite_leaves_the_step_out(kind, bad):
    ps = _params([(300,), (64, 1000)], torch.float16)
    opt = _cls(kind)(ps, **HYPER, max_grad_norm=1.0)
    _set_grads(ps, 0)
    opt.step()
    want = [p.detach().clone() for p in ps], copy.deepcopy(opt.state_dict()["state"])
    _set_grads(ps, 1)
    ps[1].grad[5, 7] = bad
    opt.step()
    assert not math.isfinite(opt.grad_norm.item())
    for p, w in zip(ps, want[0]):
        assert torch.equal(p.data, w)
    for key, st in opt.state_dict()["state"].items():
        for k, v in st.items():
            assert torch.equal(v.view(torch.uint8) if "float8" in str(v.dtype) else v,
                               want[1][key][k].view(torch.uint8) if "float8" in str(v.dtype) else want[1][key][k])
    gs = _set_grads(ps, 2)
    norm = math.sqrt(sum((g.double() ** 2).sum().item() for g in gs))
    _check_step(opt, opt.step, min(1.0, 1.0 / (norm + 1e-6)), 6 * EPS24)


@pytest.mark.parametrize("kind", ["fp32", "8bit"])
def test_a_gradient_that_is_not_finite_stays_with_its_element(kind):
    """NaN: without a clip only the element itself is lost; an infinity may cost its block of 256 the moments, no more."""
    ps, qs = _params([(2048,)], torch.float32), _params([(2048,)], torch.float32)
    a, b = _cls(kind)(ps, **HYPER), _cls(kind)(qs, **HYPER)
    for k in range(3):
        _set_grads(ps, k), _set_grads(qs, k)
        if k == 1:
            ps[0].grad[300] = math.nan
            ps[0].grad[1000] = math.inf
        a.step(), b.step()
    same = torch.ones(2048, dtype=torch.bool, device="cuda")
    same[300] = same[1000] = False
    assert not torch.isfinite(ps[0].data[[300, 1000]]).any()
    assert torch.isfinite(ps[0].data[same]).all()
    if kind == "8bit":      # moments that are no numbers are held as some
        st = a.state[ps[0]]
        assert all(torch.isfinite(st[key].float()).all() for key in ("exp_avg_q", "exp_avg_sq_q"))
    if kind == "8bit":
        same[768:1024] = False
    assert torch.equal(ps[0].data[same], qs[0].data[same])


def test_moments_in_8_bits_are_unbiased():
    """Constant gradients: v after T steps is g^2 (1 - b2^T) in the mean, although a step moves it by far less than a spacing.
    The stochastic rounding of a step has a variance below step * gain <= v/4 * v (1 - b2) for each element, so that after T
    steps the mean over n elements is off by less than 6 * v * sqrt(T (1 - b2) / 4 / n)."""
    n, steps, g = 1 << 16, 400, 0.37
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    p.grad = torch.full((n,), g, device="cuda")
    opt = _cls("8bit")([p], lr=1e-3, betas=(0.9, 0.999))
    for _ in range(steps):
        opt.step()
    st = opt.state[p]
    m, v = ref.decode(st["exp_avg_q"], st["exp_avg_scale"]).double(), ref.decode(st["exp_avg_sq_q"], st["exp_avg_sq_scale"]).double()
    want = g * g * (1 - 0.999 ** steps)
    assert abs(v.mean().item() - want) < 6 * g * g * math.sqrt(steps * 0.001 / 4 / n)
    assert abs(m.mean().item() - g) < 6 * g / 8 / math.sqrt(n) * 3
    fall = torch.zeros_like(p.grad)
    p.grad = fall
    for _ in range(400):      # and it falls again
        opt.step()
    v2 = ref.decode(st["exp_avg_sq_q"], st["exp_avg_sq_scale"]).double().mean().item()
    assert abs(v2 - want * 0.999 ** 400) < 6 * g * g * math.sqrt(800 * 0.001 / 4 / n)


@pytest.mark.parametrize("kind", ["fp32", "8bit"])
@pytest.mark.parametrize("clip", [None, 0.05])
def test_captured_steps_equal_eager_ones(kind, clip):
    """Two graphs of one optimizer, replayed in turn, with a schedule: counts and random bits go on from replay to replay."""
    pe, pg = _params(SHAPES, torch.bfloat16), _params(SHAPES, torch.bfloat16)
    oe, og = _cls(kind)(pe, **HYPER, max_grad_norm=clip), _cls(kind)(pg, **HYPER, max_grad_norm=clip)
    _set_grads(pg, 0)
    og.prime_for_cuda_graph()
    assert all(og.state[p]["step"].item() == 0 for p in pg if p.numel())
    graphs = []
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            og.step()
    for k in range(6):
        for p, g in zip(pe, _set_grads(pe, k)):
            pass
        for p, q in zip(pg, pe):
            p.grad.copy_(q.grad)
        for opt in (oe, og):
            opt.param_groups[0]["lr"] = 1e-3 * 0.5 ** k
        oe.step()
        og.update_captured_hypers()
        graphs[k % 2].replay()
        torch.cuda.synchronize()
        if clip is not None:
            assert oe.grad_norm.item() == og.grad_norm.item()
    for p, q in zip(pe, pg):
        assert torch.equal(p.data, q.data)
        if p.numel():
            assert og.state[q]["step"].item() == 6
            for key, v in oe.state[p].items():
                w = og.state[q][key]
                assert torch.equal(v.view(torch.uint8) if "float8" in str(v.dtype) else v, w.view(torch.uint8) if "float8" in str(w.dtype) else w)


@pytest.mark.parametrize("change", ["same", "moved", "lr", "scale", "none", "unaligned", "limit"])
@pytest.mark.parametrize("kind", ["fp32", "8bit"])
def test_table_equals_full_path(kind, change):
    shapes = [(64, 48), (33, 770), (300,), (512, 512)]
    (pa, pb), keep = (_params(shapes, torch.bfloat16), _params(shapes, torch.bfloat16)), []
    oa, ob = (_cls(kind)([{"params": ps[:2]}, {"params": ps[2:], "lr": 3e-3}], **HYPER, max_grad_norm=1.0 if change == "limit" else None)
              for ps in (pa, pb))
    for k in range(4):
        for ps, opt in ((pa, oa), (pb, ob)):
            old = [p.grad for p in ps]
            gs = _set_grads(ps, 10 + k)
            keep.append((old, gs))
            if change not in ("moved", "unaligned") and k:
                for p, o, g in zip(ps, old, gs):
                    if o is not None:
                        o.copy_(g)
                        p.grad = o
            if change == "none" and k == 2:
                ps[1].grad = None
            if change == "unaligned" and k == 2:
                _set_grads(ps, 10 + k, packed=True)
            if change == "lr":
                opt.param_groups[0]["lr"] = 1e-3 * 0.5 ** k
            if change == "scale":
                opt.param_groups[1]["grad_scale"] = 0.25 ** k
            if change == "limit":
                opt.max_grad_norm = [1.0, 0.01, 0.01, 2.0][k]
        oa.step()
        ob._table = None
        ob.step()
        assert oa._table is not None
    for p, q in zip(pa, pb):
        assert torch.equal(p.data, q.data)


@pytest.mark.parametrize("kind", ["fp32", "8bit"])
def test_other_streams_mixed_types_and_many_groups(kind):
    """Parameters of three types in one optimizer, 20 groups (more than travel as kernel arguments), on a side stream."""
    ps = [q for i, dt in enumerate((torch.float32, torch.bfloat16, torch.float16)) for q in _params([(100 + i,), (16, 77), (2049,)] * 3, dt, i)][:20]
    opt = _cls(kind)([{"params": [p], "lr": 1e-3 * (1 + i)} for i, p in enumerate(ps)], **{**HYPER, "lr": 1e-3}, max_grad_norm=0.02)
    side = torch.cuda.Stream()
    for k in range(2):
        for i, p in enumerate(ps):
            p.grad = _params([tuple(p.shape)], p.dtype, 50 * k + i, scale=1e-2)[0].data
        norm = math.sqrt(sum((p.grad.double() ** 2).sum().item() for p in ps))
        torch.cuda.synchronize()

        def step():
            with torch.cuda.stream(side):
                opt.step()
            side.synchronize()

        _check_step(opt, step, min(1.0, 0.02 / (norm + 1e-6)), 6 * EPS24)


def test_more_than_2_to_the_31_elements():
    import came_b200
    rows, cols = 70001, 32768      # 2.29e9
    p = torch.nn.Parameter(torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16))
    p.grad = torch.zeros_like(p)
    spots = [0, 255, 2 ** 31 - 8, 2 ** 31, 2 ** 31 + 12345, rows * cols - 300, rows * cols - 1]
    for s in spots:
        p.grad.view(-1)[s] = 0.5
    for cls in (came_b200.AdamW8bit,):
        opt = cls([p], lr=0.25, weight_decay=0.0)
        opt.step()
        norm = came_b200.clip_grad_norm_([p], math.inf)
        assert abs(norm.item() - 0.5 * math.sqrt(len(spots))) < 1e-6
        flat = p.data.view(-1)
        assert all(flat[s].item() == -0.25 for s in spots)      # the first step is lr, whatever the gradient
        assert torch.count_nonzero(flat[: 1 << 31]).item() + torch.count_nonzero(flat[1 << 31:]).item() == len(spots)
        del opt, flat


def test_runs_in_a_sharded_stepper():
    import came_b200
    from came_b200.partition import ShardedParams, ShardedStepper
    shapes = [(64, 96), (300,), (33, 7)]
    sharded = ShardedParams(shapes, torch.bfloat16, "cuda", 1, 0)
    gen = torch.Generator(device="cuda").manual_seed(3)
    for v in sharded.views:
        v.copy_(torch.randn(v.shape, device="cuda", generator=gen) * 0.02)
    ps = [torch.nn.Parameter(v) for v in sharded.views]
    _set_grads(ps, 1)
    stepper = ShardedStepper(sharded, dict(enumerate(ps)), lambda q: came_b200.AdamW8bit(q, lr=1e-3, max_grad_norm=1.0))
    (opt,) = stepper.opts
    norm = math.sqrt(sum((p.grad.double() ** 2).sum().item() for p in ps))
    _check_step(opt, stepper.step, min(1.0, 1.0 / (norm + 1e-6)), 6 * EPS24 if norm > 1 else 0.0)
    two = ShardedParams(shapes, torch.bfloat16, "cuda", 1, 0, buckets=2)
    with pytest.raises(ValueError, match="max_grad_norm"):
        ShardedStepper(two, {i: torch.nn.Parameter(v) for i, v in enumerate(two.views)},
                       lambda q: came_b200.AdamW8bit(q, lr=1e-3, max_grad_norm=1.0))


def test_training_with_all_of_them():
    """A small model: matrices under AdamW8bit, the rest under AdamW, clipped together by clip_grad_norm_, the steps of a second
    copy under one optimizer with max_grad_norm: parameters stay together, every step follows the definition."""
    import came_b200
    torch.manual_seed(0)

    def build():
        torch.manual_seed(1)
        return torch.nn.Sequential(torch.nn.Linear(64, 200), torch.nn.GELU(), torch.nn.LayerNorm(200), torch.nn.Linear(200, 10)).cuda()

    a, b = build(), build()
    mats = [p for p in a.parameters() if p.dim() == 2]
    rest = [p for p in a.parameters() if p.dim() != 2]
    o8, o32 = came_b200.AdamW8bit(mats, **HYPER), came_b200.AdamW(rest, **HYPER)
    o = came_b200.AdamW8bit(b.parameters(), **HYPER, max_grad_norm=0.1)
    for k in range(5):
        x, y = torch.randn(32, 64, device="cuda"), torch.randint(0, 10, (32,), device="cuda")
        for net in (a, b):
            net.zero_grad(set_to_none=True)
            torch.nn.functional.cross_entropy(net(x), y).backward()
        plain = [p.grad.double() for p in a.parameters()]
        want = math.sqrt(sum((g ** 2).sum().item() for g in plain))
        norm = came_b200.clip_grad_norm_(a.parameters(), 0.1)
        assert abs(norm.item() - want) <= 6 * EPS24 * want
        c = min(1.0, 0.1 / (want + 1e-6))
        for p, g in zip(a.parameters(), plain):
            assert ((p.grad.double() - g * c).abs() <= 8 * EPS24 * (g * c).abs()).all()
        _check_step(o8, o8.step)
        _check_step(o32, o32.step)
        want = math.sqrt(sum((p.grad.double() ** 2).sum().item() for p in b.parameters()))
        _check_step(o, o.step, min(1.0, 0.1 / (want + 1e-6)), 6 * EPS24)


def test_came_and_adamw_tensors_share_a_plan():
    """One tensor table with both kinds steps each as a table of its own would."""
    import came_b200
    from came_b200.engine import DevicePlan

    def make():
        ps = _params([(96, 130), (300,), (64, 256), (513,), (33, 70)], torch.bfloat16)
        _set_grads(ps, 5)
        return ps, came_b200.CAMECUDA(ps[:2], lr=1e-3, weight_decay=0.1), came_b200.AdamW8bit(ps[2:4], **HYPER, max_grad_norm=0.1), came_b200.AdamW(
            ps[4:], **HYPER, max_grad_norm=0.1)

    (pa, ca, a8, _), (pb, cb, b8, _) = make(), make()
    opts, entries, hypers = (ca, a8), [], []
    for o in opts:
        es, hs, _ = o._collect()
        for e in es:
            e.group += len(hypers)
        entries += es
        hypers += hs
    plan = DevicePlan(torch.device("cuda", 0), entries)
    for k in range(3):
        plan.step(hypers)
        cb.step(), b8.step()
        for p, q in zip(pa[:4], pb[:4]):
            assert torch.equal(p.data, q.data)
        assert plan.grad_norm.item() == b8.grad_norm.item()
    assert a8.state[pa[2]]["step"].item() == 3
    plan.close()


def test_nothing_of_adamw_is_pushed():
    """The push mode of the weight exchange does not know these tensors: they are reported as to be copied, and are not stored."""
    import came_b200
    flat = torch.zeros(8192, device="cuda", dtype=torch.bfloat16)
    p = torch.nn.Parameter(flat[:4096].view(64, 64))
    p.grad = torch.ones_like(p)
    opt = came_b200.AdamW([p], **HYPER)
    opt.prime_for_cuda_graph()
    mirror = torch.zeros_like(flat)
    opt._engine.set_push(flat.data_ptr(), flat.numel() * 2, [mirror.data_ptr()])
    (plan,) = opt._engine.plans.values()
    opt.step()
    torch.cuda.synchronize()
    assert plan.pushed() == [False] and not mirror.any() and flat[:4096].all()


@pytest.mark.parametrize("kind", ["fp32", "8bit"])
def test_the_kernels_that_run(kind):
    from tests.parity_util import kernels_of
    ps = _params([(300, 40), (77,)], torch.bfloat16)
    _set_grads(ps, 1)
    name = {"fp32": "adamw", "8bit": "adamw8"}[kind]
    for limit, names in ((None, {name}), (1.0, {name, "grad_norm"})):
        opt = _cls(kind)(ps, **HYPER, max_grad_norm=limit)
        opt.step()
        assert kernels_of(opt) == names and opt.last_step_launches == len(names)


def test_two_optimizers_on_two_streams():
    """Launches that overlap at their ends, of optimizers that have nothing to do with one another."""
    import came_b200
    sets = [_params([(500, 512), (129,), (2000, 33)], torch.bfloat16, s) for s in (1, 2, 1, 2)]
    for i, ps in enumerate(sets):
        _set_grads(ps, 10 + i % 2)
    opts = [came_b200.AdamW8bit(ps, **HYPER, max_grad_norm=0.5) for ps in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    norms = []
    for _ in range(20):
        for s, o, ps in zip(streams, opts[:2], sets[:2]):
            with torch.cuda.stream(s):
                o.step()
                norms.append(came_b200.clip_grad_norm_(ps, math.inf))
    torch.cuda.synchronize()
    for o in opts[2:]:
        for _ in range(20):
            o.step()
    torch.cuda.synchronize()
    for a, b in zip(sets[:2], sets[2:]):
        assert all(torch.equal(p.data, q.data) for p, q in zip(a, b))
    assert len({n.item() for n in norms[::2]}) == len({n.item() for n in norms[1::2]}) == 1


@pytest.mark.parametrize("kind", ["fp32", "8bit"])
def test_refusals(kind):
    p = torch.nn.Parameter(torch.zeros(8, 8, device="cuda", dtype=torch.float64))
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="float64"):
        _cls(kind)([p]).step()
    ps = _params([(8, 8), (5,)], torch.float32)
    _set_grads(ps, 0)
    opt = _cls(kind)([{"params": [torch.nn.Parameter(torch.zeros(1, device="cuda"))]} for _ in range(64)] + [{"params": ps}], lr=1e-3)
    with pytest.raises(RuntimeError, match="param_groups"):
        opt.step()
    opt = _cls(kind)(ps, lr=1e-3)
    opt.step()
    opt.param_groups[0]["betas"] = (0.9, 1.0)
    before = [q.detach().clone() for q in ps]
    with pytest.raises(ValueError, match="betas"):
        opt.step()
    assert all(torch.equal(a, b.data) for a, b in zip(before, ps))
    opt.param_groups[0]["betas"] = (0.9, 0.99)
    st = opt.state[ps[0]]
    key = "exp_avg" if kind == "fp32" else "exp_avg_q"
    st[key] = torch.zeros(3, device="cuda", dtype=st[key].dtype)
    with pytest.raises(RuntimeError, match="shape"):
        opt.prime_for_cuda_graph()
    with pytest.raises(ValueError, match="twice"), warnings.catch_warnings():
        warnings.simplefilter("ignore")
        _cls(kind)([ps[1], ps[1]]).step()
    with pytest.raises(ValueError, match="twice"):
        alias = torch.nn.Parameter(ps[1].data)
        alias.grad = ps[1].grad
        _cls(kind)([ps[1], alias]).step()
    s = torch.nn.Parameter(torch.zeros(4, 4, device="cuda"))
    s.grad = torch.sparse_coo_tensor(torch.tensor([[0], [0]]), torch.tensor([1.0]), (4, 4)).cuda()
    with pytest.raises(RuntimeError, match="sparse"):
        _cls(kind)([s]).step()


def test_eager_steps_between_replays():
    import came_b200
    pe, pg = _params([(300, 40), (77,)], torch.float32), _params([(300, 40), (77,)], torch.float32)
    oe, og = came_b200.AdamW8bit(pe, **HYPER), came_b200.AdamW8bit(pg, **HYPER)
    _set_grads(pe, 3), _set_grads(pg, 3)
    og.prime_for_cuda_graph()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        og.step()
    for k in range(6):
        oe.step()
        graph.replay() if k % 3 else og.step()
    torch.cuda.synchronize()
    assert all(torch.equal(p.data, q.data) for p, q in zip(pe, pg)) and og.state[pg[0]]["step"].item() == 6
