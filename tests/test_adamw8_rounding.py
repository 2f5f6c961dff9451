"""The rounding of AdamW8bit's moments over the whole range of its formats, subnormals included: the oracle's mean, codes held to
the definition, moments that have to die out and moments that have to grow."""
import pytest
import torch

from tests import adamw_ref as ref


def _spread(n, low, high, device="cpu", seed=0):
    """Magnitudes 2^low .. 2^high, evenly in the exponent; the first of every 256 is the largest."""
    gen = torch.Generator(device=device).manual_seed(seed)
    x = torch.exp2(torch.rand(n, generator=gen, device=device) * (high - low) + low)
    x[::256] = 1.5 * 2.0 ** high
    return x


@pytest.mark.parametrize("which", ["m", "v"])
def test_the_mean_over_many_steps_is_the_value(which):
    """A rounding to one of two neighbours u apart has a variance of u^2 / 4 at most: the mean of T = 600 is off by less than
    6 u / (2 sqrt(T)) = 0.123 u."""
    top, _, least, _, _, _ = ref.FORMATS[which]
    x = _spread(4096, -12.0 if which == "m" else -15.9, float(top))
    if which == "m":
        x[1::2] *= -1.0
    total = torch.zeros(4096, dtype=torch.float64)
    for t in range(1, 601):
        codes, scale = ref.encode(x, which, t)
        assert (scale == 1.0).all()
        total += codes.double()
    u = ref.spacing(x, which).double()
    assert ((total / 600 - x.double()).abs() <= 0.123 * u).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("level", [-140, -60, -10, 0, 13, 14, 20, 62])
def test_codes_follow_the_definition_at_any_magnitude(level, offset, dtype):
    """betas = (0, 0): the moments are g and g^2 rounded once to fp32, in blocks that span 24 powers of two around 2^level; the bytes
    equal those of the definition in 64 bits."""
    import came_b200
    n = 256 * 40 + 77
    buf = torch.zeros(n + offset, device="cuda", dtype=dtype)
    p, g = torch.nn.Parameter(buf[offset:]), torch.zeros_like(buf)[offset:]
    p.grad = g
    opt = came_b200.AdamW8bit([p], lr=1e-3, betas=(0.0, 0.0))
    for t in range(1, 4):
        x = _spread(n, level - 23.0, level + 0.4, "cuda", t)
        x[1::3] *= -1.0
        g.copy_(x)
        if t == 2:
            g[512:768] = 0.0
        opt.step()
        st, f = opt.state[p], g.float()
        for x, which, key in ((f, "m", "exp_avg"), (f * f, "v", "exp_avg_sq")):
            codes, scale = ref.encode(x, which, t)
            assert torch.equal(scale, st[key + "_scale"].float())
            assert torch.equal(codes.float(), st[key + "_q"].float()), (which, t)


@pytest.mark.gpu
def test_infinite_moments_are_held_as_finite_ones():
    import came_b200
    p = torch.nn.Parameter(torch.zeros(1024, device="cuda"))
    p.grad = _spread(1024, -3.0, 3.0, "cuda")
    p.grad[100] = 1e25      # its square is infinite
    opt = came_b200.AdamW8bit([p], betas=(0.0, 0.0))
    opt.step()
    st = opt.state[p]
    assert all(torch.isfinite(st[key].float()).all() for key in ("exp_avg_q", "exp_avg_sq_q"))
    v = ref.decode(st["exp_avg_sq_q"], st["exp_avg_sq_scale"])
    assert v[100] >= 2.0 ** 127 and torch.isfinite(p.data).all()


def _two(n, **hyper):
    import came_b200
    ps = [torch.nn.Parameter(torch.zeros(n, device="cuda")) for _ in range(2)]
    g = torch.zeros(n, device="cuda")
    for p in ps:
        p.grad = g
    return ps, g, came_b200.AdamW8bit(ps[:1], **hyper), came_b200.AdamW(ps[1:], **hyper)


@pytest.mark.gpu
@pytest.mark.parametrize("betas", [(0.9, 0.95), (0.9, 0.999)])
def test_parameters_whose_gradient_has_ended_come_to_rest(betas):
    """Half of every block gets no gradient after step 200.  Its first moments are zero 600 steps later: |y| < 2^8 falls to the least
    code 2^-9 within ln(2^17) / ln(1 / 0.9) = 112 steps or so, and from there to zero with a chance of 0.1 a step (0.9^400 = 5e-19).
    The way that is left is that of the fp32 states: a rounding of m has a standard deviation of m / 16 at most, ten of them
    in the sum 0.2; those of v add up to 0.35 of v at 0.999 (each sqrt(0.001 v * v / 4), 500 of them), 0.18 of its root, whose
    inverse is 5 % too large in the mean; the median over 1024 elements of a ratio that spreads by 0.27 is known to
    6 * 1.25 * 0.27 / 32 = 6 %."""
    n = 2048
    (p8, p32), g, o8, o32 = _two(n, lr=1e-3, betas=betas, eps=1e-12, weight_decay=0.0)
    gen = torch.Generator(device="cuda").manual_seed(5)
    ended = torch.arange(n, device="cuda") % 2 == 0
    for t in range(1, 801):
        g.copy_(torch.randn(n, generator=gen, device="cuda") * 1e-3)
        if t > 200:
            g[ended] = 0.0
        o8.step(), o32.step()
        if t == 200:
            at8, at32 = p8.detach().clone(), p32.detach().clone()
    assert not o8.state[p8]["exp_avg_q"].float()[ended].any()
    assert o8.state[p8]["exp_avg_q"].float()[~ended].count_nonzero() > 900
    way8, way32 = (p8 - at8).abs()[ended].median().item(), (p32 - at32).abs()[ended].median().item()
    assert abs(way8 / way32 - 1.0) <= 0.11 + 0.02      # (fp32 states: what is left of m counts to the end, 2 % at most)
    rest = p8.detach()[ended].clone()
    o8.step()
    assert torch.equal(p8.detach()[ended], rest)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-4, 2e-4])
def test_parameters_whose_gradient_begins_late_take_steps_of_the_right_size(size):
    """Half of every block is quiet for 1000 steps, then gets gradients of `size` times the others': second moments between one and
    forty times the least code.  The root mean square of an update is that of the fp32 states to 10 % (the inverse root of
    few codes: about 5 % too large)."""
    n = 4096
    (p8, p32), g, o8, o32 = _two(n, lr=1e-3, betas=(0.9, 0.999), eps=1e-14, weight_decay=0.0)
    gen = torch.Generator(device="cuda").manual_seed(6)
    late = torch.arange(n, device="cuda") % 2 == 0
    sums = [0.0, 0.0]
    for t in range(1, 2001):
        g.copy_(torch.randn(n, generator=gen, device="cuda") * 1e-3)
        g[late] *= size if t > 1000 else 0.0
        before = [p.detach().clone() for p in (p8, p32)] if t > 1200 else None
        o8.step(), o32.step()
        if before is not None:
            for k, p in enumerate((p8, p32)):
                sums[k] = sums[k] + ((p.detach() - before[k])[late].double() ** 2).mean()
    assert abs((sums[0] / sums[1]).sqrt().item() - 1.0) <= 0.1
