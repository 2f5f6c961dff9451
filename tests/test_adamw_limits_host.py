"""What the AdamW step and the gradient clip refuse, count and remember, on the CPU."""
import copy
import ctypes as C
import math
import pickle
import subprocess
import sys

import pytest
import torch

import came_b200
from came_b200 import _host, _lib


def test_clip_refuses_addresses_off_their_elements():
    """(the kernels take 16 bytes from the first boundary of an element on)"""
    lib = _lib.load()
    need = lib.came_b200_clip_workspace_bytes(1)

    def code(at, dtype, norm=0x1000, n=100):
        return lib.came_b200_clip_grad_norm((_lib.CameGradRef * 1)(_lib.CameGradRef(at, n, dtype, 0)), 1, 1.0, norm, 0x2000, need, None)

    for at, dtype in ((0x10001, _lib.DT_F32), (0x10002, _lib.DT_F32), (0x10001, _lib.DT_F16), (0x10003, _lib.DT_BF16)):
        assert code(at, dtype) == _lib.E_INVALID and b"aligned" in lib.came_b200_last_error()
    assert code(0x10000, _lib.DT_F32, norm=0x1002) == _lib.E_INVALID and b"aligned" in lib.came_b200_last_error()


class _Plan:
    """A plan as the engine sees it, without a device."""
    made = []

    def __init__(self, device, entries):
        self.device, self.n, self.captured, self.open, self.records, self.last_launches = device, len(entries), 0, True, None, 0
        self.structure = tuple(e.structure_key() for e in entries)
        self.addresses = tuple((e.p.data_ptr(), e.g.data_ptr()) for e in entries)
        _Plan.made.append(self)

    def repoint(self, entries):
        return self.addresses == tuple((e.p.data_ptr(), e.g.data_ptr()) for e in entries) or not self.captured

    def set_hyper(self, records):
        assert self.open
        self.records = list(records)

    def close(self):
        self.open = False


def test_a_captured_plan_is_never_closed(monkeypatch):
    """A graph reads the workspace and the page-locked records of the plan it was captured from at every replay."""
    from came_b200 import engine
    monkeypatch.setattr(engine, "DevicePlan", _Plan)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    _Plan.made = []

    def entries(flags=0):
        t = [torch.zeros(4) for _ in range(4)]
        return [engine.Entry(p=t[0], g=t[1], mode=_lib.MODE_ADAMW, flags=flags, group=0, m=t[2], sq_row=t[3], res_row=torch.zeros(()))]

    e, first = engine.StepEngine(), entries()
    e.prepare(first)
    e.prepare(entries())                      # another set: the first plan goes
    assert [p.open for p in _Plan.made] == [False, True]
    _Plan.made[1].captured = 1
    e.prepare(entries(_lib.F_ADAMW_CLIP))     # ... but not one that was captured
    e.prepare(entries())
    assert [p.open for p in _Plan.made] == [False, True, False, True]
    _Plan.made[3].captured = 2
    e.invalidate()
    assert _Plan.made[3].open and not e.plans
    e.prepare(first)
    e.set_hyper(["a", "b", "c"])              # every graph sees a schedule
    assert _Plan.made[1].records == ["a"] and _Plan.made[3].records == ["a", "b"] and _Plan.made[4].records == ["a", "b", "c"]
    _Plan.made[4].captured = 2                # (a group was added since)
    e.set_hyper(["d", "e", "f"])
    assert _Plan.made[4].records == ["d", "e"]
    _Plan.made[4].captured = 0
    assert e.last_captured() == [_Plan.made[3]]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="prime_for_cuda_graph"):
        e.prepare(entries())


def test_a_plan_whose_steps_may_still_run_is_waited_for(monkeypatch):
    """It may have been stepped on another stream than the one its workspace was allocated on."""
    from came_b200 import engine
    done = []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: done.append(device))
    monkeypatch.setattr(_Plan, "close", lambda self: done.append("closed"))
    e = engine.StepEngine()
    for launches in (0, 2):
        plan = _Plan("cuda:3", [])
        plan.last_launches = launches
        e.plans["cuda:3"] = plan
        e.invalidate()
    assert done == ["closed", "cuda:3", "closed"]


@pytest.mark.parametrize("cls", [came_b200.AdamW, came_b200.AdamW8bit])
def test_the_limit_of_a_captured_step(cls):
    """Without a limit the record's is infinite (factor 1), and a captured step cannot be switched between the two."""
    opt = cls([torch.nn.Parameter(torch.zeros(4))], max_grad_norm=5.0)
    assert opt._hypers()[0].clip_threshold == 5.0
    opt.max_grad_norm = None
    assert opt._hypers()[0].clip_threshold == math.inf and opt._table_args() == (math.inf,)

    class Plan:
        def __init__(self, clips, captured):
            self.clips, self.captured, self.records = clips, captured, None

        def set_hyper(self, records):
            self.records = records

        def close(self):
            pass

    for clips in (False, True):
        for retired in (False, True):      # (retired: an eager step has taken another plan since)
            plan, other = Plan(clips, 1), Plan(not clips, 0)
            opt._engine.retired = [plan] if retired else []
            opt._engine.plans = {"cuda": other if retired else plan}
            opt.max_grad_norm = 2.0 if clips else None
            opt.update_captured_hypers()
            assert plan.records[0].clip_threshold == (2.0 if clips else math.inf)
            plan.records = None
            opt.max_grad_norm = None if clips else 2.0
            with pytest.raises(ValueError, match="captured"):
                opt.update_captured_hypers()
            assert plan.records is None
    opt._engine.retired, opt._engine.plans = [], {}


@pytest.mark.filterwarnings("ignore:optimizer contains a parameter group with duplicate parameters")
@pytest.mark.parametrize("cls", [came_b200.AdamW, came_b200.AdamW8bit])
def test_a_parameter_listed_twice_is_refused_whatever_its_strides(cls):
    """(a step takes a copy of a parameter that is not contiguous, but its states are one)"""
    for p in (torch.nn.Parameter(torch.zeros(4, 6).t()), torch.nn.Parameter(torch.zeros(2, 3, 4, 4).to(memory_format=torch.channels_last)),
              torch.nn.Parameter(torch.zeros(5))):
        p.grad = torch.ones_like(p)
        alias = torch.nn.Parameter(p.data)
        alias.grad = p.grad
        for twice in ([p, p], [p, alias]):
            opt = cls(twice)
            with pytest.raises(ValueError, match="twice"):
                opt.step()
            assert not opt.state      # refused before anything is made
    empty = [torch.nn.Parameter(torch.zeros(0)) for _ in range(2)]
    for p in empty:
        p.grad = torch.zeros(0)
    with pytest.raises(RuntimeError, match="CUDA"):      # (empty ones share no element)
        cls(empty).step()


def _table(monkeypatch, shape, mode):
    """The row of the tensor table that DevicePlan makes of a parameter."""
    from came_b200 import engine
    rows = []

    class Lib:
        def came_b200_workspace_bytes(self, descs, n):
            rows.extend((d.rows, d.cols, d.batch) for d in descs)
            return 0

    monkeypatch.setattr(engine._lib, "load", lambda: Lib())
    monkeypatch.setattr(engine._lib, "check", lambda rc: (_ for _ in ()).throw(StopAsyncIteration))
    t = [torch.empty(shape, device="meta") for _ in range(2)]
    e = engine.Entry(p=t[0], g=t[1], mode=mode, flags=0, group=0, m=t[0], sq_row=t[0], res_row=t[0])
    with pytest.raises(StopAsyncIteration):
        engine.DevicePlan(torch.device("cpu"), [e])
    return rows[0]


def test_elements_are_counted_in_64_bits(monkeypatch):
    lib = _lib.load()
    size = lambda **kw: lib.came_b200_workspace_bytes((_lib.CameTensorDesc * 1)(_desc(**kw)), 1)  # noqa: E731
    for mode in (_lib.MODE_ADAMW, _lib.MODE_ADAMW8):
        assert size(mode=mode, rows=1 << 31, cols=0) > 0 and size(mode=mode, rows=(1 << 33) + 1, cols=0) > 0
        assert size(mode=mode, rows=4_100_000_000_000, cols=0) == 0 and size(mode=mode, rows=1 << 62, cols=1 << 62) == 0
        assert size(mode=mode, rows=1 << 62, cols=1, batch=(1 << 32) - 1) == 0
    assert size(mode=_lib.MODE_FP32, rows=1 << 31, cols=0) == 0
    with monkeypatch.context() as m:
        for shape in ((1 << 32, 2, 2), (3, 1 << 31, 1, 1), ((1 << 31) + 5,), (5, 7), ()):
            for mode in (_lib.MODE_ADAMW, _lib.MODE_ADAMW8):
                assert _table(m, shape, mode) == (math.prod(shape), 0, 0)
        assert _table(m, (3, 5, 7), _lib.MODE_FP32) == (5, 7, 3) and _table(m, (5, 7), _lib.MODE_FP32) == (5, 7, 0)
        with pytest.raises(RuntimeError, match="matrices"):
            _table(m, (1 << 32, 2, 2), _lib.MODE_FP32)


def _desc(**kw):
    d = _lib.CameTensorDesc()
    for k, f in enumerate(("p", "g", "m", "m_absmax", "sq_row", "sq_row_absmax", "res_row")):
        setattr(d, f, 0x10000 * (k + 1))
    d.rows, d.cols, d.p_dtype, d.g_dtype = 64, 64, _lib.DT_BF16, _lib.DT_BF16
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_an_empty_parameter_does_not_keep_the_table_away():
    """AdamW passes over it: it has no place in the plan, and the table has to know."""
    class Plan:
        handle = None
        addresses = ()

    def build(sizes, n, *limit):
        ps = [torch.nn.Parameter(torch.zeros(s)) for s in sizes]
        for p in ps:
            p.grad = torch.zeros_like(p)
        groups = [dict(params=ps, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)]
        keep.append(ps)
        return _host.StepTable().build(groups, [(Plan(), -1, n)], [], *limit)

    keep = []
    assert build([4], 1, 1.0) and build([4, 0], 1, 1.0) and build([0, 4, 0], 1, math.inf) and build([(3, 0, 2), 4, 5], 2, 1.0)
    assert not build([4, 0], 2, 1.0) and not build([4, 5], 1, 1.0) and not build([4, 0], 1)      # (the last: a CAME table)


def test_no_norm_before_the_first_step():
    """(prime_for_cuda_graph() makes the plan, whose norm then is a zero that nobody took)"""
    class Plan:
        grad_norm, last_launches, captured = 0.0, 0, 0

        def close(self):
            pass

    opt = came_b200.AdamW([torch.nn.Parameter(torch.zeros(4))], max_grad_norm=1.0)
    opt._engine.plans = {"cuda": Plan()}
    assert opt.grad_norm is None
    opt._engine.plans["cuda"].last_launches = 2
    assert opt.grad_norm == 0.0
    opt._engine.plans = {}


@pytest.mark.parametrize("limit", [None, 1.0, 0.37, math.inf])
def test_records_of_the_native_table_equal_those_of_the_python_path(limit):
    """Byte for byte, AdamW's one per group and CAME's two."""
    from came_b200.engine import make_adamw_hyper, make_hyper
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.zeros(4)

    class Plan:
        handle = None
        addresses = ()

    def records(groups, *args):
        table = _host.StepTable()
        assert table.build(groups, [(Plan(), -1, 1)], [], *args)
        return table.records(groups)

    ps = [[p], [], []]
    groups = [dict(params=ps[0], lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1),
              dict(params=ps[1], lr=3e-4, betas=[0.0, 0.95], eps=1e-30, weight_decay=0.0, grad_scale=1.0 / 1024),
              dict(params=ps[2], lr=0, betas=(0.95, 0.0), eps=0.0, weight_decay=1, grad_scale=3)]
    bound = math.inf if limit is None else limit
    want = b"".join(bytes(make_adamw_hyper(g["lr"], g["betas"], g["eps"], g["weight_decay"], bound, float(g.get("grad_scale", 1.0))))
                    for g in groups)
    assert records(groups, bound) == want
    opt = came_b200.AdamW([dict(g, params=[torch.nn.Parameter(torch.zeros(1))]) for g in groups], max_grad_norm=limit)
    assert b"".join(bytes(h) for h in opt._hypers()) == want
    table = _host.StepTable()
    assert table.build(groups, [(Plan(), -1, 1)], [], bound)
    assert table.records(groups * 22) is None      # (66 of 64)
    groups[1]["betas"] = (0.9, 1.0)
    assert table.records(groups) is None      # (the Python path raises)
    came = [dict(params=ps[0], lr=1e-3, betas=(0.9, 0.999, 0.9999), eps=(1e-30, 1e-16), clip_threshold=1.0, weight_decay=0.1, grad_scale=0.5)]
    want = b"".join(bytes(make_hyper(1e-3, (0.9, 0.999, 0.9999), (1e-30, 1e-16), 1.0, 0.1, python_scalars=k, grad_scale=0.5)) for k in (False, True))
    assert records(came) == want


def test_a_plan_beyond_the_hosts_memory_is_an_error():
    """4e12 elements are two billion work items: the list of them does not fit what the process may have, and no exception (which
    would end the process) leaves the C entry."""
    code = """
import ctypes as C, importlib.util, resource, sys
spec = importlib.util.spec_from_file_location("_lib", sys.argv[1])
_lib = importlib.util.module_from_spec(spec)
spec.loader.exec_module(_lib)
lib = _lib.load()
used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + (2 << 30),) * 2)
d = _lib.CameTensorDesc()
for k, f in enumerate(("p", "g", "m", "m_absmax", "sq_row", "sq_row_absmax", "res_row")):
    setattr(d, f, 0x10000 * (k + 1))
d.rows, d.cols, d.mode, d.p_dtype, d.g_dtype = 4000000000000, 0, _lib.MODE_ADAMW8, _lib.DT_BF16, _lib.DT_BF16
plan = C.c_void_p()
rc = lib.came_b200_plan_create((_lib.CameTensorDesc * 1)(d), 1, 0x10000000, 1 << 60, None, C.byref(plan))
print(rc, plan.value, lib.came_b200_last_error().decode())
"""
    out = subprocess.run([sys.executable, "-c", code, _lib.__file__], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.startswith(f"{_lib.E_INVALID} None") and "memory" in out.stdout, (out.returncode, out.stdout, out.stderr)


@pytest.mark.parametrize("name,kw", [("AdamW", dict(max_grad_norm=0.5)), ("AdamW8bit", {}), ("CAME8bit", dict(cuda_1d_runtime_mode="repeated_fp16_pairmin"))])
def test_copies_and_pickles_keep_the_settings(name, kw):
    p = torch.nn.Parameter(torch.zeros(4, 4))
    opt = getattr(came_b200, name)([p], lr=1e-3, **kw)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert other._engine is not opt._engine and other.param_groups[0]["lr"] == 1e-3 and other.last_step_launches == 0
        for key in ("_max_grad_norm", "cuda_nonfactored_use_fp16_update", "prefer_cuda_2d_fast_path"):
            assert getattr(other, key, "none") == getattr(opt, key, "none")
        other.param_groups[0]["params"][0].grad = torch.ones(4, 4)
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            other.step()
    engine = opt._engine
    opt.load_state_dict(opt.state_dict())
    assert opt._engine is engine      # (with the plans that graphs read)
