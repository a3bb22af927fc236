"""CPU checks of the AdamW operators at their edges: refusals of the row-aware gradient norm, optimiser state around a capture, floors of the 8-bit moments."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import adamw_oracle as ao


def _one(*x):
    return (ctypes.c_void_p * 1)(*x)


def test_norm_without_rows_that_are_left_alone_refuses_before_it_launches():
    from gs_icp_slam_amd import _lib
    lib = _lib.load()
    width, frozen = (ctypes.c_int * 1)(3), (ctypes.c_int * 1)(1)
    D = _lib.AdamWDevice

    def norm(d, grad=64, numel=300, dtype=0, n=1, out=64, scratch=64):
        return lib.gsicp_grad_norm_rows(n, _one(grad), (ctypes.c_longlong * 1)(numel), (ctypes.c_int * 1)(dtype), ctypes.addressof(d) if d else None, 1.0, out, 64, scratch, None)
    w, f = ctypes.addressof(width), ctypes.addressof(frozen)
    ok = dict(live_rows=64, row_width=w, row_freeze=64, group_frozen=f)
    assert norm(None) == -2
    assert norm(D(live_rows=64)) == -2                                            # no row_width
    assert norm(D(row_width=w, row_freeze=64)) == -2                              # no group_frozen
    assert norm(D(grad_rows=64, **ok)) == -2                                      # gradients that were not written
    assert norm(D(**ok), dtype=1) == -2 and norm(D(**ok), numel=1 << 32) == -2    # as in the step
    assert norm(D(**ok), numel=-1) == -2 and norm(D(**ok), numel=(1 << 33) + 1) == -2 and norm(D(**ok), dtype=3) == -2
    assert norm(D(**ok), grad=0) == -2 and norm(D(**ok), grad=1 << 58) == -2 and norm(D(**ok), out=None) == -2 and norm(D(**ok), n=-1) == -2
    assert norm(D(**ok), numel=1 << 30, scratch=None) == -2
    assert b"gsicp_grad_norm" in lib.gsicp_last_error()


@pytest.mark.parametrize("bits", [32, 8])
def test_state_made_by_the_warm_up_of_a_capture_gets_its_first_value(bits):
    """Parameters and state as a capture's warm-up leaves them, put back: a master weight that it made is the parameter, not zero."""
    from gs_icp_slam_amd.graph import MapperIterationGraph
    from gs_icp_slam_amd.optim import FusedAdamW
    params = {k: torch.nn.Parameter(torch.full((300,), v, dtype=dt)) for k, v, dt in (("a", 1.5, torch.bfloat16), ("b", -2.0, torch.float16), ("c", 3.0, torch.float32),
                                                                                    ("old", 0.25, torch.bfloat16))}
    mg = MapperIterationGraph.__new__(MapperIterationGraph)
    mg.params, mg.optimizer = params, FusedAdamW(params.values(), state_bits=bits, master_weights=True, capturable=True)
    mg.optimizer._new_state(params["old"], torch.zeros((), dtype=torch.int32) + 4)
    mg.optimizer.state[params["old"]]["master"].fill_(0.250001)
    snap_p = {k: p.detach().clone() for k, p in params.items()}
    snap_s = {p: {k: v.clone() for k, v in mg.optimizer.state.get(p, {}).items()} for p in params.values()}
    shared = torch.zeros((), dtype=torch.int32)
    with torch.no_grad():
        for k, p in params.items():
            if k != "old":
                mg.optimizer._new_state(p, shared)
            p.add_(1.0)
            for v in mg.optimizer.state[p].values():
                v.add_(1)
    mg._restore(snap_p, snap_s)
    for k, p in params.items():
        st = mg.optimizer.state[p]
        assert torch.equal(p, snap_p[k]) and int(st["step"]) == (4 if k == "old" else 0)
        assert ("master" in st) == (p.dtype != torch.float32)
        if k == "old":
            assert torch.equal(st["master"], torch.full((300,), 0.250001))
        elif k != "c":
            assert torch.equal(st["master"], p.detach().float())
        assert all(not bool(st[n].any()) for n in (("exp_avg", "exp_avg_sq") if bits == 32 else ("moments", "block_exps")))


@pytest.mark.parametrize("counts", [(7, 7, 0), (3, 5, 3)])
@pytest.mark.parametrize("adamw", [True, False])
def test_a_step_count_of_the_host_survives_a_capture(adamw, counts):
    """A state with host step counts (made without capturable, or by hand) goes to the device in the warm-up; putting it back must not lose the count."""
    from gs_icp_slam_amd.graph import MapperIterationGraph
    from gs_icp_slam_amd.optim import FusedAdam, FusedAdamW
    params = {k: torch.nn.Parameter(torch.ones(300)) for k in "abc"}
    mg = MapperIterationGraph.__new__(MapperIterationGraph)
    mg.params, mg.optimizer = params, (FusedAdamW if adamw else FusedAdam)(params.values(), capturable=True)
    for p, n in zip(params.values(), counts):
        mg.optimizer.state[p].update(step=n, exp_avg=torch.full((300,), 0.5), exp_avg_sq=torch.full((300,), 0.25))
    snap_p = {k: p.detach().clone() for k, p in params.items()}
    snap_s = {p: {k: v.clone() if torch.is_tensor(v) else v for k, v in mg.optimizer.state[p].items()} for p in params.values()}
    device_counts = {}
    for p, n in zip(params.values(), counts):
        step = device_counts.setdefault(n, torch.full((), n + 2, dtype=torch.int32))      # as two warm-up iterations leave it, shared by equal counts
        mg.optimizer.state[p].update(step=step, exp_avg=torch.full((300,), 9.0), exp_avg_sq=torch.full((300,), 9.0))
    mg._restore(snap_p, snap_s)
    for p, n in zip(params.values(), counts):
        st = mg.optimizer.state[p]
        assert int(st["step"]) == n and bool((st["exp_avg"] == 0.5).all()) and bool((st["exp_avg_sq"] == 0.25).all())


def test_an_eps_that_the_reciprocal_takes_for_zero_is_refused():
    """0 / (0 + 1e-40) is 0, 0 * (1 / 1e-40) with the subnormal taken for zero would be NaN.  The pointers are never followed."""
    from gs_icp_slam_amd import _lib
    lib = _lib.load()
    for name, tail in (("gsicp_adamw_step", (None, None, None)), ("gsicp_adamw_step_8bit", (0, None, None, None, None))):
        def call(eps, n):
            return getattr(lib, name)(n, _one(4096), _one(1 << 20), None, _one(1 << 21), _one(1 << 22), (ctypes.c_longlong * 1)(0), (ctypes.c_int * 1)(0), (ctypes.c_double * 1)(1e-3),
                                      (ctypes.c_double * 1)(0.0), 0.9, 0.999, eps, 1, *tail)
        for eps in (1e-40, 2.0 ** -127, 2.0 ** -149, 1.1754942e-38):
            assert call(eps, 1) == -2 and b"eps" in lib.gsicp_last_error(), eps


# ------------------------------------------------------------------------------------------------ state dicts of other optimisers
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("saved,loaded", [(True, True), (True, False), (False, True), (False, False)])
def test_masters_after_loading_are_those_that_the_optimiser_keeps(bits, saved, loaded):
    from gs_icp_slam_amd.optim import FusedAdamW
    dtypes = [torch.bfloat16, torch.float16, torch.float32, torch.bfloat16]
    ps = [torch.nn.Parameter(torch.randn(130).to(dt)) for dt in dtypes]
    a = FusedAdamW(ps, state_bits=bits, master_weights=saved)
    for p in ps[:3]:
        a._new_state(p, 4)
        if "master" in a.state[p]:
            a.state[p]["master"] += 1e-4
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    b = FusedAdamW(qs, state_bits=bits, master_weights=loaded)
    b.load_state_dict(a.state_dict())
    for p, q in zip(ps[:3], qs):
        st = b.state[q]
        assert ("master" in st) == (loaded and q.dtype != torch.float32)
        if "master" in st:
            assert st["master"].dtype == torch.float32 and torch.equal(st["master"], a.state[p]["master"] if saved else q.detach().float())
            assert st["master"].data_ptr() != q.data_ptr()
    assert not b.state.get(qs[3])                            # not stepped yet: the first step makes its state
    # masters of 16-bit parameters do not belong to the f32 parameters that take over their state
    wide = [torch.nn.Parameter(p.detach().float()) for p in ps]
    c = FusedAdamW(wide, state_bits=bits, master_weights=True)
    c.load_state_dict(a.state_dict())
    assert all("master" not in c.state[q] for q in wide[:3])


def test_a_state_without_weight_decay_leaves_that_of_the_groups():
    from gs_icp_slam_amd.optim import FusedAdam, FusedAdamW
    make = lambda: [{"params": [torch.nn.Parameter(torch.ones(9))]}, {"params": [torch.nn.Parameter(torch.ones(5))], "lr": 0.25}]       # noqa: E731
    a = FusedAdam(make(), lr=0.5)
    for g in a.param_groups:
        a.state[g["params"][0]].update(step=3, exp_avg=torch.ones_like(g["params"][0]), exp_avg_sq=torch.ones_like(g["params"][0]))
    groups = make()
    groups[1]["weight_decay"] = 0.3
    b = FusedAdamW(groups, lr=1.0, weight_decay=0.05)
    b.load_state_dict(a.state_dict())
    assert [g["weight_decay"] for g in b.param_groups] == [0.05, 0.3] and [g["lr"] for g in b.param_groups] == [0.5, 0.25]
    c = FusedAdamW(make(), weight_decay=0.7)
    c.load_state_dict(b.state_dict())
    assert [g["weight_decay"] for g in c.param_groups] == [0.05, 0.3]              # a state that has it says it


@pytest.mark.parametrize("cls,kw,taken", [("AdamW", {}, True), ("AdamW", dict(weight_decay=0.3), True), ("Adam", {}, True), ("Adam", dict(weight_decay=0.1), False),
                                          ("AdamW", dict(amsgrad=True), False), ("AdamW", dict(maximize=True), False), ("Adam", dict(maximize=True), False)])
def test_states_of_torch_optimisers_with_another_update_are_refused(cls, kw, taken):
    from gs_icp_slam_amd.optim import FusedAdamW
    p = torch.nn.Parameter(torch.ones(9))
    a = getattr(torch.optim, cls)([p], lr=0.125, **kw)
    p.grad = torch.ones(9)
    a.step()
    opt = FusedAdamW([torch.nn.Parameter(torch.ones(9))])
    if taken:
        opt.load_state_dict(a.state_dict())
        st = opt.state[opt.param_groups[0]["params"][0]]
        assert st["step"] == 1 and isinstance(st["step"], int) and torch.equal(st["exp_avg"], a.state[p]["exp_avg"])
        assert opt.param_groups[0]["lr"] == 0.125 and opt.param_groups[0]["weight_decay"] == a.param_groups[0]["weight_decay"]
    else:
        with pytest.raises(ValueError, match="FusedAdamW"):
            opt.load_state_dict(a.state_dict())
        assert not opt.state and opt.param_groups[0]["lr"] == 1e-3


def test_counts_of_a_torch_optimiser_that_agree_share_one_device_counter():
    """One counter per parameter would mean a launch per parameter, and no shared counter for the captured iteration to advance."""
    from gs_icp_slam_amd.optim import FusedAdamW
    ps = [torch.nn.Parameter(torch.ones(n)) for n in (5, 6, 7, 8)]
    a = torch.optim.AdamW(ps)
    for k in range(3):
        for p in ps:
            p.grad = torch.ones_like(p)
        if k == 1:
            ps[3].grad = None
        a.step()
    opt = FusedAdamW([torch.nn.Parameter(p.detach().clone()) for p in ps], capturable=True)
    opt.load_state_dict(a.state_dict())
    counters = [opt.state[p]["step"] for p in opt.param_groups[0]["params"]]
    assert [int(c) for c in counters] == [3, 3, 3, 2] and all(c.dtype == torch.int32 and c.shape == () for c in counters)
    assert len({c.data_ptr() for c in counters[:3]}) == 1 and counters[3].data_ptr() != counters[0].data_ptr()
    # counters of one's own that agree by chance stay apart: they need not agree after the next step
    b = FusedAdamW([torch.nn.Parameter(p.detach().clone()) for p in ps], capturable=True)
    own = [torch.full((), 4, dtype=torch.int32) for _ in range(2)]
    for p, c in zip(b.param_groups[0]["params"], (own[0], own[0], own[1], own[1])):
        b._new_state(p, c)
    opt.load_state_dict(b.state_dict())
    counters = [opt.state[p]["step"].data_ptr() for p in opt.param_groups[0]["params"]]
    assert counters[0] == counters[1] != counters[2] == counters[3]


@pytest.mark.parametrize("cls", ["FusedAdam", "FusedAdamW"])
def test_counters_elsewhere_are_not_handed_to_a_kernel(cls):
    """A state loaded to the host, or with torch's float counters: its address is not one that the loss kernel or the step may advance."""
    from gs_icp_slam_amd import optim
    params = [torch.nn.Parameter(torch.ones(3, device="meta")) for _ in range(3)]
    opt = getattr(optim, cls)(params, capturable=True)
    there = torch.zeros((), dtype=torch.int32, device="meta")
    for step, taken in ((there, True), (torch.zeros((), dtype=torch.int32), False), (torch.zeros((), device="meta"), False), (torch.tensor(4.0), False), (4, False)):
        for p in params:
            opt.state[p]["step"] = step
        assert (opt.shared_step_tensor() is there) == taken, step
        assert all(optim._counts_beside(opt.state[p]["step"], p) == taken for p in params)
    host = torch.full((), 6, dtype=torch.int32)
    q = torch.nn.Parameter(torch.ones(3, dtype=torch.float64))
    made = {}
    a, b = optim._counter_beside(host, params[0], made), optim._counter_beside(host, params[1], made)
    assert a is b and a.dtype == torch.int32 and a.device.type == "meta"
    assert optim._counter_beside(host.clone(), params[0], made) is not a                       # another counter that agrees by chance
    c = [optim._counter_beside(x, q, made) for x in (6, torch.tensor(6.0), 7)]
    assert c[0] is c[1] is not c[2] and [int(x) for x in c] == [6, 6, 7]


# ------------------------------------------------------------------------------------------------ lists of tensors
def test_written_lists_raise_their_version_counters():
    from gs_icp_slam_amd import _tensor_lists
    a, b, c = [torch.zeros(2), torch.zeros(0)], (torch.zeros(3),), [None, torch.zeros(1)]
    version = lambda: [t._version for t in (*a, *b, c[1])]           # noqa: E731
    _tensor_lists.wrote((b"", a, b, c), 0b101)
    assert version() == [1, 1, 0, 1]
    _tensor_lists.wrote((b"", a, b, c), 0b010)
    assert version() == [1, 1, 1, 1]
    with torch.inference_mode():
        still = torch.zeros(2)                                       # counts no versions
    _tensor_lists.wrote((b"", [still]), 1)
    for args in ((), ((b"", a),), ((b"", a), -1), ([b"", a], 1), ((b"", a), "x")):
        with pytest.raises(TypeError):
            _tensor_lists.wrote(*args)


# ------------------------------------------------------------------------------------------------ the floors of 8-bit moments
def test_an_element_at_a_floor_moves_by_at_most_three_times_the_largest_step():
    """m / sqrt(v) of what the codes stand for, in blocks whose small elements have the same ratio as the large one, or any."""
    rng = np.random.default_rng(0)
    worst = 0.0
    for k in range(400):
        m, v = np.empty(128, np.float32), np.empty(128, np.float32)
        if k < 100:                                      # the largest first moment just above a power of two, its second just below one, the rest far below
            m[0], v[0] = 2.0 ** -5, 1.99 * 2.0 ** -9
            scale = 2.0 ** -rng.uniform(14.5, 16.0)
            m[1:], v[1:] = m[0] * scale, v[0] * scale ** 2
        else:
            m[:] = rng.choice([-1, 1], 128) * np.exp(rng.uniform(-14, 0, 128))
            v[:] = (m.astype(np.float64) * np.exp(rng.uniform(-2, 2, 128))) ** 2
        codes, exps = ao.encode(m, v, *ao.random_bits(128, 3, k + 1, 0))
        a, b = ao.decode(codes, exps)
        ratio = np.abs(a) / np.sqrt(b)
        floor = (codes & 127 == 1) | (codes >> 8 == 1)
        if floor.any():
            worst = max(worst, ratio[floor].max() / ratio.max(where=~floor, initial=0.0))
    assert 2.0 < worst <= 3.0 * (1 + 1e-12), worst
