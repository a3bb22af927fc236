"""CPU checks around the AdamW operators: the 8-bit format's restatement (unbiased rounding, ends of the range), the refusals of the C ABI (before anything is launched) and
of the Python layer, and the state dict."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import adamw_oracle as ao


def test_random_bits_are_uniform_and_unbiased_per_element():
    steps = 400
    um, uv = np.zeros((steps, 512)), np.zeros((steps, 512))
    for t in range(steps):
        um[t], uv[t] = (x / 65536.0 for x in ao.random_bits(512, 3, t + 1, 2))
    for u in (um, uv):
        assert abs(u.mean() - 0.5 + 2.0 ** -17) < 6 / np.sqrt(12 * u.size)
        assert np.abs(u.mean(0) - 0.5).max() < 6 / np.sqrt(12 * steps)              # each element over the steps
        assert np.abs(u.mean(1) - 0.5).max() < 6 / np.sqrt(12 * 512)                # each step over the elements
        assert abs(np.corrcoef(u[0], u[1])[0, 1]) < 6 / np.sqrt(512)
    assert np.abs((um - 0.5).mean(0) @ (uv - 0.5).mean(0)) < 1.0
    assert not np.array_equal(ao.random_bits(64, 3, 1, 0)[0], ao.random_bits(64, 3, 1, 1)[0])
    a, b = ao.random_bits(512, 3, 1, 2)
    c, d = ao.random_bits(128, 3, 1, 2, first=256)
    assert np.array_equal(a[256:384], c) and np.array_equal(b[256:384], d)


def test_rounding_to_codes_is_unbiased_and_within_one_code():
    rng = np.random.default_rng(0)
    n, reps = 256, 4096
    v = np.exp(rng.uniform(np.log(1e-9), 0, n)).astype(np.float32)               # all inside the 30 exponents of a block
    m = (rng.choice([-1, 1], n) * np.exp(rng.uniform(np.log(3e-6), 0, n))).astype(np.float32)      # and below the smallest code of the first moments
    sm, sv = np.zeros(n), np.zeros(n)
    for t in range(reps):
        codes, exps = ao.encode(m, v, *ao.random_bits(n, 1, t + 1, 0))
        a, b = ao.decode(codes, exps)
        low = np.repeat(1.125 * 2.0 ** ((exps & 255).astype(int) - 127), 128)
        assert (np.abs(b - v) <= v / 8).all()
        assert (np.abs(a - m) <= np.maximum(np.abs(m) / 8, low)).all()
        sm += a
        sv += b
    # spacing of the codes is at most an eighth: the mean of `reps` roundings is within 6 standard errors of the value, and the 16 random bits' grain
    assert (np.abs(sv / reps - v) <= 6 * (v / 16) / np.sqrt(reps) + v * 2.0 ** -18).all()
    assert (np.abs(sm / reps - m) <= 6 * np.maximum(np.abs(m) / 16, np.sqrt(np.abs(m) * low)) / np.sqrt(reps) + low * 2.0 ** -16).all()


def test_a_slow_average_moves_where_nearest_rounding_would_not():
    """b2 = 0.999: a step changes v by a thousandth, codes are 6 to 12 % apart.  The mean over many elements follows the average exactly, to its statistical error."""
    n, steps, b2 = 4096, 1500, 0.999
    v = np.full(n, 1.0, dtype=np.float32)
    truth = 1.0
    exps = None
    for t in range(steps):
        codes, exps = ao.encode(np.zeros(n, dtype=np.float32), (np.float32(b2) * v).astype(np.float32), np.zeros(n), ao.random_bits(n, 5, t + 1, 0)[1])
        v = ao.decode(codes, exps, np.float32)[1]
        truth *= b2
    # relative variance added per step <= 0.001 * (1/8)^2; after `steps` of them < 0.16: six standard errors of the mean of 4096 elements
    assert abs(v.mean() / truth - 1) < 6 * np.sqrt(0.001 / 64 * steps * 10) / np.sqrt(n)


def test_ends_of_the_range():
    n = 128
    u = ao.random_bits(n, 0, 1, 0)
    v = np.zeros(n, dtype=np.float32)
    m = np.zeros(n, dtype=np.float32)
    v[0], v[1], v[2], v[3] = np.finfo(np.float32).max, 1e-38, 1e-45, np.inf
    m[0], m[1], m[2], m[3] = -np.finfo(np.float32).max, np.nan, -np.inf, 1e-45
    codes, exps = ao.encode(m, v, *u)
    a, b = ao.decode(codes, exps)
    assert exps[0] == (240 | 224 << 8) and (codes[4:] == 0).all()
    assert abs(b[0] / float(v[0]) - 1) <= 1 / 8 and b[1] == b[2] == 1.125 * 2.0 ** 97 and np.isinf(b[3])         # above zero stays above zero
    assert abs(a[0] / float(m[0]) - 1) <= 1 / 8 and np.isnan(a[1]) and np.isnan(a[2]) and a[3] == 0
    for k in range(64):          # never rounded up to infinity
        c, e = ao.encode(m, v, *ao.random_bits(n, k, 1, 0))
        a, b = ao.decode(c, e, np.float32)
        assert np.isfinite(a[0]) and np.isfinite(b[0])
    codes, exps = ao.encode(np.zeros(n, dtype=np.float32), np.full(n, 1e-45, dtype=np.float32), *u)
    assert exps[0] == (1 | 1 << 8) and (codes == 1 << 8).all()


def test_gathered_rows_keep_their_values():
    rng = np.random.default_rng(0)
    rows, width = 500, 5
    m = (rng.normal(size=rows * width) * np.exp(3 * rng.normal(size=rows * width))).astype(np.float32)
    v = (rng.normal(size=rows * width) ** 2 * np.exp(6 * rng.normal(size=rows * width))).astype(np.float32)
    m[::7], v[::11], m[3], v[4] = 0, 0, np.nan, np.inf
    codes, exps = ao.encode(m, v, *ao.random_bits(rows * width, 1, 1, 0))
    a, b = ao.decode(codes, exps)
    index = np.concatenate([np.flatnonzero(rng.random(rows) < 0.6), [3, 3, -1, rows, 0]])
    c2, e2 = ao.gather(codes, exps, width, index, rows)
    a2, b2 = ao.decode(c2, e2)
    inside = (index >= 0) & (index < rows)
    want = [np.where(inside[:, None], x.reshape(rows, width)[np.where(inside, index, 0)], 0.0).reshape(-1) for x in (a, b)]
    low = lambda shift: np.repeat(1.125 * 2.0 ** ((e2.astype(int) >> shift & 255) - 127), 128)[:c2.size]      # noqa: E731
    for got, w, lo, floor in ((a2, want[0], low(0), 0.0), (b2, want[1], low(8), None)):
        small = (np.abs(w) < lo) & (w != 0)
        np.testing.assert_array_equal(got[~small], w[~small])
        np.testing.assert_array_equal(got[small], lo[small] if floor is None else 0.0)
    assert np.array_equal(ao.gather(*ao.gather(codes, exps, width, np.arange(rows), rows), width, np.arange(rows), rows)[0], ao.gather(codes, exps, width, np.arange(rows), rows)[0])


def _arrays(n, **kw):
    d = dict(params=[4096 * (k + 1) for k in range(n)], grads=[1 << 20] * n, masters=None, s0=[(1 << 21) + 4096 * k for k in range(n)], s1=[(1 << 22) + 4096 * k for k in range(n)],
             numel=[100] * n, dtype=[0] * n, lr=[1e-3] * n, wd=[0.0] * n)
    d.update(kw)
    ptr = lambda x: None if x is None else (ctypes.c_void_p * len(x))(*x)       # noqa: E731
    return [n, ptr(d["params"]), ptr(d["grads"]), ptr(d["masters"]), ptr(d["s0"]), ptr(d["s1"]), (ctypes.c_longlong * n)(*d["numel"]) if d["numel"] else None,
            (ctypes.c_int * n)(*d["dtype"]), None if d["lr"] is None else (ctypes.c_double * n)(*d["lr"]), (ctypes.c_double * n)(*d["wd"])]


def test_c_abi_refuses_before_it_launches():
    """Every call below is refused by the host checks; the pointers are never followed."""
    from gs_icp_slam_amd import _lib
    lib = _lib.load()

    def step(n=2, betas=(0.9, 0.999), eps=1e-8, t=1, dev=None, eight=False, **kw):
        a = _arrays(n, **kw) + [betas[0], betas[1], eps, t]
        if eight:
            return lib.gsicp_adamw_step_8bit(*a, 0, None, None, dev, None)
        return lib.gsicp_adamw_step(*a, None, dev, None)
    D = _lib.AdamWDevice
    width = (ctypes.c_int * 2)(3, 3)
    for eight in (False, True):
        assert step(eight=eight, numel=[100, -1]) == -2 and step(eight=eight, numel=[100, (1 << 33) + 1]) == -2
        assert step(eight=eight, dtype=[0, 3]) == -2 and step(eight=eight, dtype=[-1, 0]) == -2
        for name in ("params", "grads", "s0", "s1"):
            assert step(eight=eight, **{name: None}) == -2
            assert step(eight=eight, **{name: [4096, 0]}) == -2
        assert step(eight=eight, params=[4096, 4096]) == -2 and step(eight=eight, params=[4096, 4100]) == -2           # the same one, an overlap
        assert step(eight=eight, s0=[4096, 1 << 21]) == -2                                                             # a moment inside a parameter
        assert step(eight=eight, grads=[4096, 1 << 20]) == -2 and step(eight=eight, grads=[(1 << 21) + 4, 1 << 20]) == -2            # a gradient inside what is written
        assert step(eight=eight, masters=[1 << 23, 0]) == -2                                                           # f32 with a master
        assert step(eight=eight, betas=(1.0, 0.999)) == -2 and step(eight=eight, betas=(0.9, -0.1)) == -2 and step(eight=eight, betas=(float("nan"), 0.9)) == -2
        assert step(eight=eight, eps=-1.0) == -2 and step(eight=eight, eps=float("nan")) == -2
        assert step(eight=eight, t=0) == -2 and step(eight=eight, lr=None) == -2
        for d in (D(), D(lr_dev=64), D(step_dev=64), D(lr_dev=64, step_dev=64, bump_step=3), D(lr_dev=64, step_dev=64, grad_rows=64),
                  D(lr_dev=64, step_dev=64, row_freeze=64, row_width=ctypes.addressof(width))):
            assert step(eight=eight, dev=ctypes.addressof(d)) == -2
        d = D(lr_dev=64, step_dev=64, grad_rows=64, row_width=ctypes.addressof(width))
        assert step(eight=eight, dev=ctypes.addressof(d), dtype=[0, 1]) == -2 and step(eight=eight, dev=ctypes.addressof(d), numel=[100, 1 << 32]) == -2
    d = D(lr_dev=64, step_dev=64, row_freeze=64, group_frozen=ctypes.addressof(width), row_width=ctypes.addressof(width))
    assert step(eight=True, dev=ctypes.addressof(d)) == -2
    assert b"gsicp_adamw_step_8bit" in lib.gsicp_last_error()
    assert lib.gsicp_adamw_step(-1, *[None] * 9, 0.9, 0.999, 1e-8, 1, None, None, None) == -2 and lib.gsicp_adamw_decode(-1, *[None] * 5, 0, None) == -2
    one = lambda *x: (ctypes.c_void_p * 1)(*x)              # noqa: E731
    k = (ctypes.c_longlong * 1)
    assert lib.gsicp_adamw_decode(1, one(64), one(64), one(64), one(0), k(5), 0, None) == -2
    assert lib.gsicp_adamw_decode(1, one(64), one(64), one(64), one(64), k(5), 2, None) == -2
    assert lib.gsicp_adamw_decode(1, one(64), one(64), one(64), one(64), k(-5), 0, None) == -2
    gather = lambda c, x, oc, ox, w, index, n, src: lib.gsicp_adamw_gather_rows(1, one(c), one(x), one(oc), one(ox), k(w), index, n, src, None)      # noqa: E731
    assert gather(1 << 12, 1 << 20, 1 << 21, 1 << 22, 3, None, 5, 9) == -2 and gather(1 << 12, 1 << 20, 0, 1 << 22, 3, 64, 5, 9) == -2
    assert gather(1 << 12, 1 << 20, 1 << 12, 1 << 22, 3, 64, 5, 9) == -2 and gather(1 << 12, 1 << 20, (1 << 12) + 52, 1 << 22, 3, 64, 5, 9) == -2       # in place, into the last row
    assert gather(1 << 12, 1 << 20, 1 << 21, 1 << 22, 3, 64, (1 << 32) // 3 + 1, 9) == -2 and gather(1 << 12, 1 << 20, 1 << 21, 1 << 22, -1, 64, 5, 9) == -2
    assert gather(1 << 12, 1 << 20, 1 << 21, 1 << 22, 3, 64, -5, 9) == -2 and gather(1 << 12, 1 << 20, 1 << 21, 1 << 22, 3, 64, 5, -9) == -2
    assert lib.gsicp_grad_norm(1, one(64), k(5), (ctypes.c_int * 1)(0), 0.0, None, 64, 64, None) == -2
    assert lib.gsicp_grad_norm(1, one(64), k(5), (ctypes.c_int * 1)(5), 0.0, 64, 64, 64, None) == -2
    assert lib.gsicp_grad_norm(1, one(0), k(5), (ctypes.c_int * 1)(0), 0.0, 64, 64, 64, None) == -2
    assert lib.gsicp_grad_norm(1, one(1 << 58), k(5), (ctypes.c_int * 1)(0), 0.0, 64, 64, 64, None) == -2
    assert lib.gsicp_grad_norm(1, one(64), k((1 << 33) + 1), (ctypes.c_int * 1)(0), 0.0, 64, 64, 64, None) == -2
    assert lib.gsicp_grad_norm(1, one(64), k(1 << 30), (ctypes.c_int * 1)(0), 0.0, 64, 64, None, None) == -2          # a large set needs its scratch
    size = lambda n, each: lib.gsicp_grad_norm_scratch_bytes(n, (ctypes.c_longlong * n)(*[each] * n), (ctypes.c_int * n)(*[0] * n))      # noqa: E731
    assert size(1, 5) == size(64, 7) == 0 and size(65, 7) == size(1, 1 << 30) > 0 and size(241, 7) > size(240, 7)


def test_python_layer_has_no_cpu_path_and_refuses_bad_options():
    from gs_icp_slam_amd.gaussian_store import GaussianStore
    from gs_icp_slam_amd.optim import FusedAdamW, adamw_step, adamw_step_8bit, decode_moments, grad_norm
    z = torch.zeros
    i16 = dict(dtype=torch.int16)
    for f in (lambda: adamw_step([z(8)], [z(8)], [z(8)], [z(8)], lr=1e-3, step=1), lambda: adamw_step_8bit([z(8)], [z(8)], [z(8, **i16)], [z(1, **i16)], lr=1e-3, step=1),
              lambda: decode_moments([z(8, **i16)], [z(1, **i16)]), lambda: grad_norm([z(8)])):
        with pytest.raises(RuntimeError):
            f()
    p = torch.nn.Parameter(z(8))
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-0.1), dict(betas=(0.9, 1.0)), dict(max_grad_norm=0.0), dict(max_grad_norm=float("nan"))):
        with pytest.raises(ValueError):
            FusedAdamW([p], **kw)
    p.grad = z(8)
    with pytest.raises(RuntimeError):
        FusedAdamW([p]).step()
    with pytest.raises(RuntimeError):
        FusedAdamW([p]).step(step_already_bumped=True)
    store = GaussianStore(16, device="cpu")
    lrs = dict.fromkeys(("xyz", "f_dc", "f_rest", "opacity", "scaling", "rotation"), 1e-3)
    with pytest.raises(RuntimeError):
        store.attach(FusedAdamW, lrs, state_bits=8)
    assert store.optimizer is None
    with pytest.raises(ValueError):
        GaussianStore(16, device="cpu", moment_bits=16)
    small = GaussianStore(16, n_rest=2, device="cpu", moment_bits=8)
    for cls, kw in ((FusedAdamW, {}), (torch.optim.Adam, {})):
        with pytest.raises(RuntimeError):
            small.attach(cls, lrs, **kw)
    opt = small.attach(FusedAdamW, lrs, state_bits=8)
    assert all(opt.state[q]["moments"].shape == q.shape and opt.state[q]["block_exps"].numel() == -(-q.numel() // 128) for q in small.params.values())
    opt = store.attach(FusedAdamW, lrs, weight_decay=0.1)
    assert all(opt.state[q]["step"] == 0 and opt.state[q]["exp_avg"].shape == q.shape for q in store.params.values())
    assert all(g["weight_decay"] == 0.1 for g in opt.param_groups)
    opt.add_param_group({"params": [p], "name": "extra"})
    assert opt.param_groups[-1]["weight_decay"] == 0.1


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_state_dict_keeps_dtypes_and_shared_counters(bits, dtype):
    from gs_icp_slam_amd.optim import FusedAdamW
    ps = [torch.nn.Parameter(torch.randn(n).to(dtype)) for n in (5, 300, 0)]
    a = FusedAdamW(ps, state_bits=bits, master_weights=True, capturable=True)
    shared = torch.full((), 7, dtype=torch.int32)
    for p in ps:
        a._new_state(p, shared)
        for k, t in a.state[p].items():
            if k != "step":
                t.random_(0, 100)
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    b = FusedAdamW(qs, state_bits=bits, master_weights=True, capturable=True)
    b.load_state_dict(a.state_dict())
    for p, q in zip(ps, qs):
        assert set(a.state[p]) == set(b.state[q])
        for k, t in a.state[p].items():
            u = b.state[q][k]
            assert t.dtype == u.dtype and torch.equal(t, u) and (t.numel() == 0 or t.data_ptr() != u.data_ptr()), k
    assert len({b.state[q]["step"].data_ptr() for q in qs}) == 1
    c = FusedAdamW([torch.nn.Parameter(p.detach().clone()) for p in ps], state_bits=bits, master_weights=True)
    c.load_state_dict(a.state_dict())
    assert all(st["step"] == 7 and isinstance(st["step"], int) for st in c.state.values())
    with pytest.raises(ValueError):
        FusedAdamW(qs, state_bits=40 - bits).load_state_dict(a.state_dict())
