"""AdamW on the CPU: constructor, records, validation in the library, the native step table with an AdamW group, and refusals."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import came_b200
from came_b200 import _host, _lib
from came_b200.engine import make_adamw_hyper
from tests import adamw_ref as ref


def test_constructor():
    w = [torch.nn.Parameter(torch.zeros(4, 4))]
    for cls in (came_b200.AdamW, came_b200.AdamW8bit):
        for bad in (dict(lr=-1.0), dict(lr=math.nan), dict(betas=(0.9, 1.0)), dict(betas=(-0.1, 0.9)), dict(betas=(0.9, 0.99, 0.999)),
                    dict(eps=-1.0), dict(weight_decay=-1.0), dict(max_grad_norm=0.0), dict(max_grad_norm=math.nan), dict(lr=torch.tensor(1.0))):
            with pytest.raises(ValueError):
                cls(w, **bad)
        opt = cls(w)
        g = opt.param_groups[0]
        assert (g["lr"], g["betas"], g["eps"], g["weight_decay"]) == (1e-3, (0.9, 0.999), 1e-8, 1e-2)
        assert opt.max_grad_norm is None and opt.grad_norm is None
        w[0].grad = torch.ones(4, 4)
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            opt.step()
        w[0].grad = None


def test_records():
    h = make_adamw_hyper(1e-3, (0.9, 0.999), 1e-8, 0.1, 2.0, 0.5)
    f = np.float32
    assert h.om_beta2 == f(1.0 - 0.999) and h.eps0 == f(1e-8) and h.clip_threshold == 2.0 and h.grad_scale == 0.5 and h.wd_lr == f(1e-4)
    assert abs((float(h.om_beta3) + float(h.reserved[1])) / math.log(0.999) - 1.0) < 2.0 ** -45
    assert abs((float(h.beta3) + float(h.reserved[0])) / math.log(0.9) - 1.0) < 2.0 ** -45
    z = make_adamw_hyper(1e-3, (0.0, 0.5), 1e-8, 0.0)
    assert z.beta3 == -math.inf and z.reserved[0] == 0.0 and z.clip_threshold == 1.0
    for betas in ((0.9, 1.0), (0.9,), (math.nan, 0.9)):
        with pytest.raises(ValueError):
            make_adamw_hyper(1e-3, betas, 1e-8, 0.0)


def _desc(**kw):
    d = _lib.CameTensorDesc()
    for k, f in enumerate(("p", "g", "m", "m_absmax", "sq_row", "sq_row_absmax", "res_row")):
        setattr(d, f, 0x10000 * (k + 1))
    d.rows, d.cols, d.mode, d.p_dtype, d.g_dtype = 64, 64, _lib.MODE_ADAMW8, _lib.DT_BF16, _lib.DT_BF16
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_validation_without_gpu():
    lib = _lib.load()
    size = lambda *ds: lib.came_b200_workspace_bytes((_lib.CameTensorDesc * len(ds))(*ds), len(ds))  # noqa: E731
    assert size(_desc()) > 0 and size(_desc(mode=_lib.MODE_ADAMW, m_absmax=None, sq_row_absmax=None)) > 0
    assert size(_desc(rows=1, cols=0)) > 0 and size(_desc(batch=5)) > 0
    for bad in (dict(m_absmax=None), dict(sq_row_absmax=None), dict(res_row=None), dict(sq_row=None), dict(m=None), dict(rows=0),
                dict(mode=5), dict(rows=(1 << 31) - 1, cols=(1 << 31) - 1), dict(g_dtype=3)):
        assert size(_desc(**bad)) == 0, bad
        assert lib.came_b200_last_error()
    handle = C.c_void_p()
    two = (_lib.CameTensorDesc * 2)(_desc(flags=_lib.F_ADAMW_CLIP), _desc())
    assert lib.came_b200_plan_create(two, 2, 0x10000000, 1 << 30, None, C.byref(handle)) == _lib.E_INVALID
    assert b"CLIP" in lib.came_b200_last_error()
    # the work lists: with fake pointers and no GPU the call gets past them and fails at its first CUDA call
    for ds in ([_desc()], [_desc(rows=5, cols=0), _desc(mode=_lib.MODE_ADAMW, g_dtype=0), _desc(rows=4096, cols=11008)],
               [_desc(flags=_lib.F_ADAMW_CLIP), _desc(rows=1, cols=0, mode=_lib.MODE_ADAMW, flags=_lib.F_ADAMW_CLIP)]):
        arr = (_lib.CameTensorDesc * len(ds))(*ds)
        rc = lib.came_b200_plan_create(arr, len(ds), 0x10000000, 1 << 40, None, C.byref(handle))
        assert rc in (_lib.E_CUDA, _lib.OK) and b"overflow" not in lib.came_b200_last_error()
    assert lib.came_b200_plan_norm_offset(None) == -1


def test_clip_validation_without_gpu():
    lib = _lib.load()
    ref1 = _lib.CameGradRef(0x10000, 100, _lib.DT_F32, 0)
    one = lambda **kw: (_lib.CameGradRef * 1)(_lib.CameGradRef(**{**dict(g=0x10000, n=100, dtype=0, reserved=0), **kw}))  # noqa: E731
    need = lib.came_b200_clip_workspace_bytes(1)
    assert 0 < need <= lib.came_b200_clip_workspace_bytes(5000) and lib.came_b200_clip_workspace_bytes(-1) == 0
    ok = dict(grads=(_lib.CameGradRef * 1)(ref1), n=1, limit=1.0, norm=0x1000, ws=0x2000, size=need)
    for bad, code in ((dict(grads=None), -1), (dict(limit=-1.0), -1), (dict(limit=math.nan), -1), (dict(norm=None), -1), (dict(n=-1), -1),
                      (dict(ws=None), -2), (dict(ws=0x2004), -2), (dict(size=need - 1), -2), (dict(grads=one(g=None)), -1),
                      (dict(grads=one(n=-1)), -1), (dict(grads=one(dtype=7)), -1), (dict(grads=one(n=1 << 50)), -4)):
        a = {**ok, **bad}
        assert lib.came_b200_clip_grad_norm(a["grads"], a["n"], a["limit"], a["norm"], a["ws"], a["size"], None) == code, bad


def test_clip_refusals_on_the_cpu():
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        came_b200.clip_grad_norm_([p], 1.0)
    with pytest.raises(TypeError):
        came_b200.clip_grad_norm_([object()], 1.0)
    assert came_b200.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0).item() == 0.0


def test_table_with_an_adamw_group():
    class Plan:
        memory = C.create_string_buffer(1 << 16)
        handle = None
        addresses = ()

    ps = [torch.nn.Parameter(torch.zeros(4, 4))]
    ps[0].grad = torch.zeros(4, 4)
    groups = [dict(params=ps, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)]
    table = _host.StepTable()
    assert table.build(groups, [(Plan(), -1, 1)], [], 1.0)
    assert table.step(groups) == -1      # the plan is closed


def test_clip_is_refused_where_an_optimizer_holds_a_part():
    from came_b200.partition import ShardedParams, ShardedStepper
    two = ShardedParams([(8, 8), (8, 8)], torch.float32, "cpu", 1, 0, buckets=2)
    make = lambda q: came_b200.AdamW(q, max_grad_norm=1.0)  # noqa: E731
    ps = {i: torch.nn.Parameter(v) for i, v in enumerate(two.views)}
    with pytest.raises(ValueError, match="max_grad_norm"):
        ShardedStepper(two, ps, make)
    stepper = ShardedStepper(two, ps, lambda q: came_b200.AdamW(q))
    stepper.opts[0].max_grad_norm = 1.0
    with pytest.raises(ValueError, match="max_grad_norm"):
        stepper.step()


def test_float8_rounding_of_the_oracle():
    """The oracle's own rounding: unbiased, within a spacing, zero blocks zero, v never to zero."""
    gen = torch.Generator().manual_seed(0)
    x = torch.rand(256 * 64, generator=gen) * torch.exp(torch.randn(256 * 64, generator=gen) * 3)
    for which in ("m", "v"):
        y, s = ref.encode(x, which, 5)
        d = ref.decode(y, s)
        step = ref.spacing(ref.blocks(x) / s[:, None], which) * s[:, None]
        assert ((d - x).abs() <= step.reshape(-1) * 1.02).all()
        same = torch.full((256 * 256,), 1.1)
        mean = sum(ref.decode(*ref.encode(same, which, t)).double().mean() for t in range(8)) / 8
        spread = 1.1 / 4 / math.sqrt(8 * 256 * 256)
        assert abs(mean - 1.1) < 6 * spread
        z, s = ref.encode(torch.zeros(300), which, 1)
        assert not z.float().any()
    lone = torch.zeros(256)
    lone[0] = 1.0
    y, s = ref.encode(lone, "v", 1)
    assert (ref.decode(y, s) > 0).all()
