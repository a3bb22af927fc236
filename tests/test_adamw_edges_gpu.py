"""The AdamW operators where they meet each other and the rest of the framework: clipping beside rows that are no parameters, masters under a capture; lists; autograd; types side by side."""
import numpy as np
import pytest
import torch

from gs_icp_slam_amd import synth
from oracle import adamw_oracle as ao
from tests.util import make_settings, torch_inputs

pytestmark = pytest.mark.gpu


def _randn(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen)


# ------------------------------------------------------------------------------------------------ clipping, live rows, frozen rows
TAILS = [(3,), (1, 3), (15, 3), (1,), (4,), (2,), (7,), (0,), (129,)]


@pytest.mark.parametrize("live,bits,freeze", [(None, 32, True)] + [(live, bits, freeze) for live in ("none", "some", "all") for bits, freeze in ((32, True), (32, False), (8, False))])
@pytest.mark.parametrize("rows,times", [(1, 1), (37, 1), (37, 15), (2777, 1), (300_007, 1)])
def test_rows_that_are_no_parameters_do_not_count_in_the_norm(rows, times, live, bits, freeze):
    """Their gradients are NaN: neither the norm nor a row that moves may see them.  Against a twin that has zeros there and no masks."""
    from gs_icp_slam_amd.optim import FusedAdamW
    gen = torch.Generator(device="cuda").manual_seed(rows + times)
    tails = [t for t in TAILS if rows < 10_000 or t != (129,)] * times
    ps = [_randn(gen, rows, *t) for t in tails] + [torch.ones((), device="cuda")]
    groups = lambda q: [{"params": [p], "name": str(i % len(TAILS)) if p.dim() else "scalar"} for i, p in enumerate(q)]       # noqa: E731
    a_p, b_p = ([torch.nn.Parameter(p.clone()) for p in ps] for _ in range(2))
    a, b = (FusedAdamW(groups(q), lr=1e-2, weight_decay=0.1, capturable=True, state_bits=bits, max_grad_norm=0.1, seed=3) for q in (a_p, b_p))
    n_live = {None: rows, "none": 0, "some": rows * 2 // 3, "all": rows}[live]
    if live is not None:
        a.set_live_rows(torch.tensor([n_live], dtype=torch.int32, device="cuda"))
    frozen = (torch.rand(rows, device="cuda", generator=gen) < 0.4)
    if freeze:
        a.set_row_freeze(frozen.to(torch.int32), ("0", "1", "2", "3", "5", "8"))
    for k in range(3):
        total, skip = 0.0, []
        for i, (p, q) in enumerate(zip(a_p, b_p)):
            g = _randn(gen, *p.shape) * 0.1
            out = torch.zeros(p.shape[0] if p.dim() else 1, dtype=torch.bool, device="cuda")
            if p.dim():
                out[n_live:] = True
                if freeze and i % len(TAILS) in (0, 1, 2, 3, 5, 8):
                    out |= frozen
            skip.append(out)
            p.grad, q.grad = g.clone(), g.clone()
            if p.dim():
                p.grad[out], q.grad[out] = float("nan"), 0.0
            total += float((q.grad.double() ** 2).sum())
        before = [p.detach().clone() for p in a_p]
        a.step()
        b.step()
        want = np.sqrt(total)
        assert abs(float(a.last_grad_norm) - want) <= 2.0 ** -24 * 1.0001 * want, (k, float(a.last_grad_norm), want)      # rounded once
        assert torch.equal(a.last_grad_norm, b.last_grad_norm)
        for i, (p, q, out) in enumerate(zip(a_p, b_p, skip)):
            with torch.no_grad():
                if p.dim():
                    assert torch.equal(p[out], before[i][out]), (k, i)
                    q[out] = before[i][out]                     # the twin decays them
                assert torch.equal(p, q), (k, i)
            if p.dim() and bits == 32:
                for n in ("exp_avg", "exp_avg_sq"):
                    assert torch.equal(a.state[p][n], b.state[q][n]), (k, i, n)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_clipped_step_follows_the_live_count(bits):
    """One graph while the live count changes on the device, gradients behind it NaN; replays between eager work, against the host form over the live rows alone."""
    from gs_icp_slam_amd.optim import FusedAdamW
    gen = torch.Generator(device="cuda").manual_seed(5)
    rows = 5000
    shapes = [(rows, 3), (rows, 45), (rows, 1)]
    p = [torch.nn.Parameter(_randn(gen, *s)) for s in shapes]
    opt = FusedAdamW(p, lr=1e-2, capturable=True, state_bits=bits, max_grad_norm=0.5)
    live = torch.tensor([3000], dtype=torch.int32, device="cuda")
    opt.set_live_rows(live)
    static = [torch.zeros_like(q) for q in p]
    for q, g in zip(p, static):
        q.grad = g
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    norm = opt.last_grad_norm
    for n in (3000, 1, 5000, 0, 4321):
        live.fill_(n)
        new = [_randn(gen, *s) for s in shapes]
        for g, x in zip(static, new):
            g.copy_(x)
            g[n:] = float("nan")
        before = [q.detach().clone() for q in p]
        torch.randn(1 << 20, device="cuda").sum().item()
        graph.replay()
        torch.cuda.synchronize()
        want = np.sqrt(sum(float((x[:n].double() ** 2).sum()) for x in new))
        assert abs(float(norm) - want) <= 2.0 ** -24 * 1.0001 * want, n
        for q, x in zip(p, before):
            assert bool(torch.isfinite(q).all()) and torch.equal(q[n:], x[n:]) and (n == 0 or not torch.equal(q[:n], x[:n])), n


@pytest.mark.parametrize("adamw", [True, False])
def test_a_parameter_without_rows_in_a_frozen_group(adamw):
    """A 0-dim parameter has no row to freeze: it moves, the frozen rows beside it do not."""
    from gs_icp_slam_amd.optim import FusedAdam, FusedAdamW
    p, scalar = torch.nn.Parameter(torch.ones(6, 2, device="cuda")), torch.nn.Parameter(torch.ones((), device="cuda"))
    opt = (FusedAdamW if adamw else FusedAdam)([{"params": [p, scalar], "name": "xyz"}], lr=0.1, capturable=True)
    frozen = torch.tensor([1, 0, 0, 1, 0, 1], dtype=torch.int32, device="cuda")
    opt.set_row_freeze(frozen, ("xyz",))
    p.grad, scalar.grad = torch.ones_like(p), torch.ones_like(scalar)
    opt.step()
    moved = (p != 1).all(1)
    assert moved.tolist() == (frozen == 0).tolist() and float(scalar.detach()) < 1.0
    with pytest.raises(RuntimeError):
        opt.set_row_freeze(frozen[:5].clone(), ("xyz",))
        opt.step()


# ------------------------------------------------------------------------------------------------ the captured mapper iteration
def _mapper(P, W, H):
    """-> (raw parameters of a map in f32, view settings, colour and depth images of a map that differs from it)."""
    from diff_gaussian_rasterization import GaussianRasterizer
    cfg = dict(synth.REPLICA)
    cam = synth.make_camera(W, H, cfg["fx"] * W / cfg["W"], cfg["fy"] * H / cfg["H"], synth.DEFAULT_POSE_A)
    g = synth.s_map(P, seed=5)
    raw = {"means3D": torch.from_numpy(g["means3D"]), "scales": torch.log(torch.from_numpy(g["scales"])), "rotations": torch.from_numpy(g["rotations"]),
           "opacities": torch.logit(torch.from_numpy(g["opacities"]).clamp(1e-4, 1 - 1e-4)), "shs": torch.from_numpy(g["shs"])}
    rs = make_settings(cam, [0.0, 0.0, 0.0])
    t2 = torch_inputs(synth.s_map(P, seed=5, perturb_seed=7))
    with torch.no_grad():
        depth, color, _, _ = GaussianRasterizer(rs)(means3D=t2["means3D"], means2D=torch.zeros_like(t2["means3D"]), shs=t2["shs"], opacities=t2["opacities"],
                                                    scales=t2["scales"], rotations=t2["rotations"])
    return raw, cam, rs, color, depth


MAPPER_LRS = {"means3D": 4e-6, "shs": 2.5e-3, "opacities": 0.05, "scales": 5e-3, "rotations": 1e-3}


@pytest.mark.parametrize("bits", [32, 8])
def test_masters_that_a_capture_makes_start_at_their_parameters(bits):
    """16-bit parameters with masters and no step before the capture, dense gradients because of the clipping."""
    from gs_icp_slam_amd.graph import MapperIterationGraph
    from gs_icp_slam_amd.optim import FusedAdamW
    W, H = 320, 200
    raw, cam, rs, color, depth = _mapper(20000, W, H)
    half = ("shs", "opacities")
    params = {k: v.cuda().to(torch.bfloat16 if k in half else torch.float32).contiguous().requires_grad_(True) for k, v in raw.items()}
    opt = FusedAdamW([{"params": [params[k]], "lr": lr} for k, lr in MAPPER_LRS.items()], lr=0.0, eps=1e-15, weight_decay=0.0, capturable=True, state_bits=bits,
                     master_weights=True, max_grad_norm=1e-3)
    mg = MapperIterationGraph(params, opt, H, W, cam["tanfovx"], cam["tanfovy"], sh_degree=0, capacity=2_000_000, warmup=2)
    mg.set_view(rs.viewmatrix, rs.projmatrix, rs.campos, color, depth)
    start = {k: p.detach().clone() for k, p in params.items()}
    mg.capture()
    for k, p in params.items():
        assert torch.equal(p, start[k])
        assert k not in half or torch.equal(opt.state[p]["master"], start[k].float())
    for n in (1, 2, 3):
        mg.set_view(rs.viewmatrix, rs.projmatrix, rs.campos, color, depth)
        assert np.isfinite(float(mg.step()))
        torch.cuda.synchronize()
    assert int(opt.state[params["means3D"]]["step"]) == 3
    for k in half:
        p, w = params[k].detach(), opt.state[params[k]]["master"]
        assert torch.equal(w.bfloat16(), p) and not torch.equal(w, start[k].float())
        # step t moves an element by at most lr sqrt(t) with exact moments (Cauchy-Schwarz over the weights of m and v); 8-bit codes are within an eighth of the moments
        # and an element at their floors moves by at most three times its block's largest step: 4 lr sqrt(t) holds for both
        assert (w - start[k].float()).abs().max() <= MAPPER_LRS[k] * (1 + 2 ** 0.5 + 3 ** 0.5) * 4, k
    mg.release()


# ------------------------------------------------------------------------------------------------ lists of tensors
def test_tensors_that_are_negated_lazily_are_refused():
    """The imaginary part of a conjugate holds the other sign in memory."""
    from gs_icp_slam_amd.optim import FusedAdamW, adamw_step, grad_norm
    g = torch.conj(torch.tensor([1 + 2j], device="cuda")).imag
    assert g.is_neg() and g.is_contiguous() and float(g) == -2.0
    new = lambda: torch.zeros(1, device="cuda")              # noqa: E731
    p, m, v = new(), new(), new()
    for lists in (([p], [g], [m], [v]), ([g], [p], [m], [v]), ([p], [m], [g], [v])):
        with pytest.raises(RuntimeError, match="negated"):
            adamw_step(*lists, lr=0.1, step=1)
    q = torch.nn.Parameter(new())
    q.grad = g
    with pytest.raises(RuntimeError, match="negated"):
        FusedAdamW([q]).step()
    with pytest.raises(RuntimeError, match="negated"):
        grad_norm([g])
    assert float(p) == float(m) == float(v) == 0.0
    adamw_step([p], [g.resolve_neg()], [m], [v], lr=0.1, step=1)
    assert float(m) < 0 < float(p)


def test_the_smallest_eps_beside_elements_without_a_gradient():
    from gs_icp_slam_amd.optim import adamw_step
    p, g, m, v = torch.full((300,), 3.0, device="cuda"), torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
    g[::7] = 1e-3
    adamw_step([p], [g], [m], [v], lr=0.5, step=1, eps=2.0 ** -126, weight_decay=0.0)
    assert bool((p[g == 0] == 3.0).all()) and bool(((p[g != 0] - 2.5).abs() <= 8 * 2.0 ** -24 * 2.5).all())
    with pytest.raises(RuntimeError, match="eps"):
        adamw_step([p], [g], [m], [v], lr=0.5, step=2, eps=1e-40)


@pytest.mark.parametrize("step", [1 << 31, (1 << 32) + 1, 1 << 40, 0, -1])
def test_step_counts_that_do_not_fit_are_refused(step):
    from gs_icp_slam_amd.optim import adamw_step, adamw_step_8bit, new_moments_8bit
    lists = [[torch.ones(5, device="cuda")] for _ in range(4)]
    with pytest.raises(RuntimeError, match="step"):
        adamw_step(*lists, lr=0.1, step=step)
    m, x = new_moments_8bit(lists[0][0])
    with pytest.raises(RuntimeError, match="step"):
        adamw_step_8bit(*lists[:2], [m], [x], lr=0.1, step=step)
    assert all(bool((t[0] == 1).all()) for t in lists)


# ------------------------------------------------------------------------------------------------ autograd
@pytest.mark.parametrize("which", ["adamw_step", "adamw_step_8bit", "FusedAdamW", "FusedAdamW capturable", "FusedAdamW masters", "FusedAdam", "FusedAdam capturable"])
def test_a_backward_over_what_a_step_has_written_is_refused(which):
    """As after torch's optimisers: the product saved the parameter, the step changed it."""
    from gs_icp_slam_amd.optim import FusedAdam, FusedAdamW, adamw_step, adamw_step_8bit, new_moments_8bit
    dtype = torch.bfloat16 if "masters" in which else torch.float32
    p = torch.nn.Parameter(torch.ones(9, device="cuda", dtype=dtype))
    other = torch.nn.Parameter(torch.ones(9, device="cuda", dtype=dtype))
    p.grad = torch.ones_like(p)
    loss = (p * other).sum()
    version = p.grad._version
    if which == "adamw_step":
        adamw_step([p], [p.grad], [torch.zeros_like(p)], [torch.zeros_like(p)], lr=0.1, step=1)
    elif which == "adamw_step_8bit":
        m, x = new_moments_8bit(p)
        adamw_step_8bit([p], [p.grad], [m], [x], lr=0.1, step=1)
    elif "AdamW" in which:
        FusedAdamW([p], capturable="capturable" in which, master_weights="masters" in which).step()
    else:
        FusedAdam([p], capturable="capturable" in which).step()
    assert p.grad._version == version
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    (p * other).sum().backward()                                     # of the new values


def test_a_step_over_inference_tensors():
    from gs_icp_slam_amd.optim import adamw_step
    with torch.inference_mode():
        lists = [[torch.full((5,), x, device="cuda")] for x in (1.0, 1.0, 0.0, 0.0)]
        adamw_step(*lists, lr=0.1, step=1)
    adamw_step(*lists, lr=0.1, step=2)
    assert bool((lists[0][0] < 0.9).all())


# ------------------------------------------------------------------------------------------------ types side by side, the device form with 16 bits and masters
SIZES = [0, 1, 2, 7, 63, 127, 128, 129, 255, 256, 257, 1000, 2049, 5003] * 5        # more tensors than a launch takes
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def _f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def _snapshot(params, grads, first, second, masters):
    return [[None if t is None else t.detach().clone() for t in ts] for ts in (params, grads, first, second, masters)]


def _check(before, after, bits, lr, wd, t, seed, device=False, clip=1.0):
    """One step of every tensor against the oracle.  device: bias corrections in float32 — 1 - b^t within 8 units of 2^-24 (the rounded exponent 1, the hardware's 2^x and its argument
    6, the difference 1), its reciprocal, the learning rate and their product 4, the reciprocal root of the other 6: 20 units of the update with all."""
    for k, (p0, g, s0, s1, w0) in enumerate(zip(*before)):
        n = p0.numel()
        if n == 0:
            continue
        p1, n0, n1, w1 = after[0][k], after[2][k], after[3][k], after[4][k]
        m, v = (_f64(s0), _f64(s1)) if bits == 32 else ao.decode(s0.cpu().numpy(), s1.cpu().numpy())
        start = _f64(p0 if w0 is None else w0)
        (P, M, V), (dp, dm, dv) = ao.step64(start, m, v, _f64(g), lr[k], wd[k], (0.9, 0.999), 1e-15, t, clip)
        if device:
            dp = dp + 20 * 2.0 ** -24 * np.abs(P - start * (1 - lr[k] * wd[k])) + 2.0 ** -24 * np.abs(P)
        if bits == 32:
            assert (np.abs(_f64(n0) - M) <= dm).all() and (np.abs(_f64(n1) - V) <= dv).all(), (t, k)
        else:
            codes, exps = ao.encode(*ao.step32(m, v, _f64(g), (0.9, 0.999)), *ao.random_bits(n, seed, t, k))
            assert np.array_equal(n0.cpu().numpy().view(np.uint16), codes) and np.array_equal(n1.cpu().numpy().view(np.uint16), exps), (t, k)
        if w0 is None:
            assert (np.abs(_f64(p1) - P) <= dp + HALF[p1.dtype] * (np.abs(P) + dp) + TINY[p1.dtype]).all(), (t, k)
        else:
            assert (np.abs(_f64(w1) - P) <= dp).all() and torch.equal(w1.to(p1.dtype), p1), (t, k)


def _grads(gen, params):
    return [(torch.randn(p.shape, device="cuda", generator=gen) * 1e-2 * (torch.rand(p.shape, device="cuda", generator=gen) < 0.7)).to(p.dtype) for p in params]


@pytest.mark.parametrize("bits", [32, 8])
def test_types_side_by_side_with_masters_for_some(bits):
    """f32, bf16 and f16 parameters in one list, every other 16-bit one with a master."""
    from gs_icp_slam_amd.optim import adamw_step, adamw_step_8bit, new_moments_8bit
    gen = torch.Generator(device="cuda").manual_seed(bits)
    dtypes = [(torch.float32, torch.bfloat16, torch.float16)[k % 3] for k in range(len(SIZES))]
    masters = [torch.randn(n, device="cuda", generator=gen) if dt != torch.float32 and k % 2 else None for k, (n, dt) in enumerate(zip(SIZES, dtypes))]
    params = [torch.randn(n, device="cuda", generator=gen).to(dt) if w is None else w.to(dt) for n, dt, w in zip(SIZES, dtypes, masters)]
    if bits == 32:
        first, second = ([torch.zeros(n, device="cuda") for n in SIZES] for _ in range(2))
    else:
        first, second = (list(x) for x in zip(*(new_moments_8bit(p) for p in params)))
    lr, wd = [10.0 ** -(2 + k % 3) for k in range(len(SIZES))], [(0.0, 0.1)[k % 2] for k in range(len(SIZES))]
    for t in (1, 2, 3):
        grads = _grads(gen, params)
        before = _snapshot(params, grads, first, second, masters)
        if bits == 32:
            adamw_step(params, grads, first, second, lr=lr, step=t, eps=1e-15, weight_decay=wd, masters=masters)
        else:
            adamw_step_8bit(params, grads, first, second, lr=lr, step=t, seed=21, eps=1e-15, weight_decay=wd, masters=masters)
        _check(before, (params, grads, first, second, masters), bits, lr, wd, t, 21)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("master", [False, True])
def test_the_device_form_with_16_bit_parameters(bits, dtype, master):
    """Eager steps, the first of which makes the masters, then replays of one captured step with eager work between."""
    from gs_icp_slam_amd.optim import FusedAdamW
    gen = torch.Generator(device="cuda").manual_seed(bits)
    params = [torch.nn.Parameter(torch.randn(n, device="cuda", generator=gen).to(dtype)) for n in SIZES]
    groups = [{"params": params[:30], "lr": 1e-2, "weight_decay": 0.1}, {"params": params[30:], "lr": 1e-4, "weight_decay": 0.0}]
    opt = FusedAdamW(groups, eps=1e-15, capturable=True, state_bits=bits, master_weights=master, seed=8)
    lr, wd = [1e-2] * 30 + [1e-4] * 40, [0.1] * 30 + [0.0] * 40
    static = [torch.zeros_like(p) for p in params]
    for p, g in zip(params, static):
        p.grad = g
    names = ("exp_avg", "exp_avg_sq") if bits == 32 else ("moments", "block_exps")
    lists = lambda: [params, static] + [[opt.state[p].get(n) for p in params] for n in names + ("master",)]       # noqa: E731
    graph = None
    for t in range(1, 7):
        for g, new in zip(static, _grads(gen, params)):
            g.copy_(new)
        if t == 1:
            made = [p.detach().clone() for p in params]
            opt.step()
            zero = [torch.zeros_like(opt.state[p][names[0]]) for p in params], [torch.zeros_like(opt.state[p][names[1]]) for p in params]
            before = [made, static, *zero, [p.float() if master else None for p in made]]
        else:
            before = _snapshot(*lists())
            if t >= 3 and graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    opt.step()
            if t == 2 or t == 5:
                opt.step()
            else:
                torch.randn(1 << 18, device="cuda").sum().item()
                graph.replay()
                torch.cuda.synchronize()
        assert int(opt.state[params[0]]["step"]) == t
        _check(before, lists(), bits, lr, wd, t, 8, device=True)


@pytest.mark.parametrize("cls", ["FusedAdam", "FusedAdamW"])
@pytest.mark.parametrize("counter", ["int32 on the host", "float32 on the host", "float32 beside", "number"])
def test_a_state_whose_counter_is_elsewhere_continues(cls, counter, tmp_path):
    """Checkpoints are loaded to the host, torch's optimisers count in float32: the capturable step moves the counter beside the parameter and goes on."""
    from gs_icp_slam_amd import optim
    gen = torch.Generator(device="cuda").manual_seed(1)
    start = [torch.randn(n, device="cuda", generator=gen) for n in (5, 300, 4001)]
    feeds = [[torch.randn(p.shape, device="cuda", generator=gen) for p in start] for _ in range(4)]

    def go(opt, params, ks):
        for k in ks:
            for p, g in zip(params, feeds[k]):
                p.grad = g.clone()
            opt.step()
    a_p = [torch.nn.Parameter(p.clone()) for p in start]
    a = getattr(optim, cls)(a_p, lr=1e-2, capturable=True)
    go(a, a_p, (0, 1))
    torch.save(a.state_dict(), tmp_path / "s.pt")
    state = torch.load(tmp_path / "s.pt", map_location="cpu" if "host" in counter else "cuda", weights_only=True)
    b_p = [torch.nn.Parameter(p.detach().clone()) for p in a_p]
    b = getattr(optim, cls)(b_p, lr=1e-2, capturable=True)
    b.load_state_dict(state)
    for p in b_p:
        st = b.state[p]
        st["step"] = {"int32 on the host": torch.full((), 2, dtype=torch.int32), "float32 on the host": torch.tensor(2.0), "float32 beside": torch.tensor(2.0, device="cuda"),
                      "number": 2}[counter]
    assert b.shared_step_tensor() is None
    go(a, a_p, (2, 3))
    go(b, b_p, (2, 3))
    for p, q in zip(a_p, b_p):
        assert torch.equal(p, q) and torch.equal(a.state[p]["exp_avg_sq"], b.state[q]["exp_avg_sq"])
        assert b.state[q]["step"].device == q.device and b.state[q]["step"].dtype == torch.int32 and int(b.state[q]["step"]) == 4


@pytest.mark.parametrize("first_steps", [0, 2])
def test_a_refused_capture_leaves_fused_adam_as_it_was(first_steps):
    """Neither a first step nor the first one after host step counts can be captured; an eager step afterwards starts from where the state stood."""
    from gs_icp_slam_amd.optim import FusedAdam
    start = [torch.ones(n, device="cuda") for n in (5, 700)]
    host, dev = ([torch.nn.Parameter(p.clone()) for p in start] for _ in range(2))
    a, b = FusedAdam(host, lr=1e-2), FusedAdam(dev, lr=1e-2, capturable=True)
    for p in host:
        p.grad = torch.full_like(p, 0.5)
    for _ in range(first_steps):
        a.step()
    for p, q in zip(host, dev):
        q.data.copy_(p)
        q.grad = p.grad.clone()
        if first_steps:
            b.state[q].update({n: v.clone() if torch.is_tensor(v) else v for n, v in a.state[p].items()})
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="outside graph capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            b.step()
    assert all(b.state[q].get("step", 0) == first_steps for q in dev)
    a.step()
    b.step()
    for p, q in zip(host, dev):
        assert torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"]) and torch.equal(a.state[p]["exp_avg_sq"], b.state[q]["exp_avg_sq"])
        assert int(b.state[q]["step"]) == first_steps + 1 == a.state[p]["step"]


# ------------------------------------------------------------------------------------------------ the functions in a graph, large gathers
def test_the_functions_in_one_captured_graph():
    """Norm, clipped 8-bit and 32-bit step, values and rows of the moments: replays against the same calls made eagerly, with eager work between."""
    from gs_icp_slam_amd.optim import adamw_step, adamw_step_8bit, decode_moments, gather_moments_8bit, grad_norm
    gen = torch.Generator(device="cuda").manual_seed(2)
    shapes = [(2001, 3), (2001, 45), (2001, 1)]
    start = [torch.randn(s, device="cuda", generator=gen) for s in shapes]
    index = torch.randint(-1, 2001, (1500,), device="cuda", generator=gen)

    def state():
        f32 = lambda: [torch.zeros(s, device="cuda") for s in shapes]      # noqa: E731
        return dict(p=[t.clone() for t in start], q=[t.clone() for t in start], g=f32(), m=f32(), v=f32(), c=[torch.zeros(s, dtype=torch.int16, device="cuda") for s in shapes],
                    x=[torch.zeros(-(-t.numel() // 128), dtype=torch.int16, device="cuda") for t in start])

    def run(s):
        n0 = grad_norm(s["g"])
        n1 = adamw_step_8bit(s["p"], s["g"], s["c"], s["x"], lr=1e-2, step=7, seed=3, max_norm=0.3)
        n2 = adamw_step(s["q"], s["g"], s["m"], s["v"], lr=1e-2, step=7, max_norm=0.3)
        m, v = decode_moments(s["c"], s["x"])
        gc, gx = gather_moments_8bit(s["c"], s["x"], index)
        return [n0, n1, n2, *m, *v, *gc, *gx]
    a, b = state(), state()
    run(b)                                       # loads the kernels
    b = state()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(b)
    for k in range(5):
        for g, h in zip(a["g"], b["g"]):
            g.copy_(torch.randn(g.shape, device="cuda", generator=gen))
            h.copy_(g)
        want = run(a)
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(want, out)), k
        assert all(torch.equal(x, y) for name in a for x, y in zip(a[name], b[name])), k


def test_gathered_rows_past_two_to_the_31():
    """As many elements as a gather takes (2^32 - 1 less what is missing to a whole row), the first and last blocks and those around 2^31."""
    from gs_icp_slam_amd.optim import gather_moments_8bit
    w = 3
    rows = (1 << 32) // w                                    # 2^32 - 1 elements
    rng = np.random.default_rng(0)
    n = rows * w
    windows = [0, (1 << 31) // 384 * 384, (n - 384) // 384 * 384]
    c = torch.zeros(n, dtype=torch.int16, device="cuda")
    x = torch.zeros(-(-n // 128), dtype=torch.int16, device="cuda")
    want = []
    for at in windows:
        codes, exps = ao.encode(rng.normal(size=384).astype(np.float32), rng.normal(size=384).astype(np.float32) ** 2, *ao.random_bits(384, 1, 1, 0))
        c[at: at + 384] = torch.from_numpy(codes.view(np.int16)).cuda()
        x[at // 128: at // 128 + 3] = torch.from_numpy(exps.view(np.int16)).cuda()
        want.append(ao.gather(codes, exps, w, np.arange(128), 128))
    index = torch.arange(rows, device="cuda")
    (oc,), (ox,) = gather_moments_8bit([c.view(rows, w)], [x], index)
    oc = oc.view(-1)
    for at, (codes, exps) in zip(windows, want):
        assert np.array_equal(oc[at: at + 384].cpu().numpy().view(np.uint16), codes), at
        assert np.array_equal(ox[at // 128: at // 128 + 3].cpu().numpy().view(np.uint16), exps), at
    assert sum(int((t != 0).sum()) for t in oc.split(1 << 28)) == sum(int((codes != 0).sum()) for codes, _ in want)
    with pytest.raises(RuntimeError):
        gather_moments_8bit([c.view(rows, w)], [x], torch.arange(rows + 1, device="cuda"))
