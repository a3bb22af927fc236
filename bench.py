#!/usr/bin/env python
"""bench.py — GS-ICP-SLAM hot path on MI355X.

One "step" = one SLAM frame's worth of the hot path on synthetic Replica-shaped input:
  tracker : pygicp.FastGICP  set_input_source + set_source_filter + align + get_source_correspondence           [REF mp_Tracker.py:191-231]
            on the S-pair exactly as SURVEY §8(d) words it (room centre, looking +z, 1 deg about y + 2 cm along x; 8 280 points, gate
            0.02 m) — `config.workload` states the motion and the LM iteration count; the second pair (corner-facing, 0.36 deg / 8.5 mm,
            inside the convergence basin) is timed as a leg
  mapper  : one full optimisation iteration — activations, GaussianRasterizer forward, the mapping loss
            0.8 L1 + 0.2 (1-SSIM) + 0.1 L1(depth/10), backward, Adam step over the parameter groups, zero_grad; P = 300 000 surfels,
            1200x680                                                                                             [REF mp_Mapper.py:219-248]
The two halves run concurrently, as the reference's two processes do [REF gs_icp_slam.py:121-131]: inside a timed block the tracker thread
runs its --steps frames and the main thread its --steps mapper iterations, each at its own pace (the reference's Tracker.run and
Mapper.run never wait for each other per frame); the block ends when both are done.  `--lockstep` joins them after every step instead
(round 1's loop; reported as a leg).
With N > 1 GPUs the mapper's tiles are sharded across ranks (strong scaling; gs_icp_slam_amd/sharded.py) and the tracker runs as a
replica on every rank (it does not shard — DESIGN.md).

Timing: `--repeats` back-to-back blocks, each EXACTLY `--steps` steps bracketed by barrier + torch.cuda.synchronize() on both sides
(max over ranks); `value` is all timed steps over all timed seconds (the mean block).  Rank 0 prints ONE JSON line with `roofline` (SURVEY §8(d) byte model over hipEvent kernel
time), `cpu_baseline` (the OpenMP GICP oracle on this host's cores) and `legs`: each half alone, both tracker pairs, the mapper iteration
launched eagerly, and `dropin_reference_loop` — what the UNMODIFIED mp_Mapper.py executes on top of the drop-in rasteriser (torch
activations, synchronous forward, torch l1/ssim, torch.optim.Adam).
"""
import argparse
import json
import os
import statistics
import sys
import time

import numpy as np

ROOT = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, ROOT)

HBM_PEAK_GBS = 8000.0   # MI355X_MICROARCH.md: HBM3E 8.0 TB/s spec
LRS = {"means3D": 1.6e-6 * 2.5, "shs": 2.5e-3, "opacities": 0.05, "scales": 5e-3, "rotations": 1e-3}   # REF arguments/__init__.py:141-148


# ---- what unmodified mp_Mapper.py runs between render_3 and optimizer.step() [REF utils/loss_utils.py:17-69; mp_Mapper.py:225-240]
def _torch_window(channel, device):
    import torch
    from math import exp
    g = torch.tensor([exp(-(x - 11 // 2) ** 2 / float(2 * 1.5 ** 2)) for x in range(11)])
    g = (g / g.sum()).unsqueeze(1)
    return g.mm(g.t()).float().unsqueeze(0).unsqueeze(0).expand(channel, 1, 11, 11).contiguous().to(device)


def _torch_l1(x, gt):
    import torch
    loss = torch.abs(x - gt)
    return torch.where(gt != 0, loss, torch.zeros_like(loss)).mean()


def _torch_ssim(img, gt, window):
    import torch
    import torch.nn.functional as F
    img = torch.where(gt != 0, img, torch.zeros_like(img))
    c = img.size(-3)
    conv = lambda t: F.conv2d(t, window, padding=5, groups=c)   # noqa: E731
    mu1, mu2 = conv(img), conv(gt)
    mu1_sq, mu2_sq, mu12 = mu1.pow(2), mu2.pow(2), mu1 * mu2
    s1, s2, s12 = conv(img * img) - mu1_sq, conv(gt * gt) - mu2_sq, conv(img * gt) - mu12
    C1, C2 = 0.01 ** 2, 0.03 ** 2
    return (((2 * mu12 + C1) * (2 * s12 + C2)) / ((mu1_sq + mu2_sq + C1) * (s1 + s2 + C2))).mean()


def _measure_pmc_traffic(kernel_substr, timeout=120.0):
    """HBM-side traffic of one kernel, MEASURED IN THIS RUN: two child runs of this script (mapper half only, a few steps) under
    `rocprofv3 --pmc FETCH_SIZE --kernel-trace` and `--pmc WRITE_SIZE --kernel-trace` — separate passes, never combined with other trace
    domains (MI355X_MICROARCH.md) — and the mean counter value per launch of the kernel x 1024 (the counters are KiB).  Returns
    (dict, None) or (None, reason).  Raw counters: the calibration of profiles/r03_pmc_calibration.json applies (FETCH_SIZE counts a wide
    coalesced stream at 0.5x and a gather of 48-byte records at 1.55x of the bytes requested; WRITE_SIZE 1.0x / 1.28x)."""
    import csv
    import shutil
    import subprocess
    import tempfile
    exe = shutil.which("rocprofv3") or "/opt/rocm/bin/rocprofv3"
    if not os.path.exists(exe):
        return None, "rocprofv3 not found"
    out = {}
    tmp = tempfile.mkdtemp(prefix="gsicp_pmc_", dir="/tmp")
    env = dict(os.environ, TMPDIR="/tmp", GSICP_BENCH_CHILD="1")
    for k in ("WORLD_SIZE", "RANK", "LOCAL_RANK"):
        env.pop(k, None)
    try:
        for counter in ("FETCH_SIZE", "WRITE_SIZE"):
            d = os.path.join(tmp, counter)
            cmd = [exe, "--pmc", counter, "--kernel-trace", "--output-format", "csv", "-d", d, "-o", "p", "--", sys.executable, os.path.abspath(__file__),
                   "--only", "mapper", "--steps", "8", "--warmup", "2", "--repeats", "1", "--views", "2", "--min-seconds", "0", "--no-cpu-baseline", "--no-legs", "--legs-file", "/tmp/gsicp_bench_legs_pmc_child.json"]
            pr = subprocess.run(cmd, cwd="/tmp", env=env, capture_output=True, text=True, timeout=timeout)
            if pr.returncode != 0:
                return None, f"rocprofv3 --pmc {counter} exited with {pr.returncode}: {pr.stderr[-300:]}"
            tot, n = 0.0, 0
            for root, _dirs, files in os.walk(d):
                for f in files:
                    if f.endswith("counter_collection.csv"):
                        for row in csv.DictReader(open(os.path.join(root, f))):
                            if kernel_substr in row["Kernel_Name"] and row["Counter_Name"] == counter:
                                tot += float(row["Counter_Value"]); n += 1
            if n == 0:
                return None, f"no {counter} rows for {kernel_substr}"
            out[counter] = tot / n * 1024.0
            out[counter + "_launches"] = n
    except Exception as e:   # noqa: BLE001 — a profiler hiccup must not take the benchmark line with it
        return None, f"{type(e).__name__}: {e}"
    finally:
        shutil.rmtree(tmp, ignore_errors=True)
    return out, None


def trained_map_leg(dev, steps=100, reps=3, n_views=8, cache=None):
    """legs.mapper_trained_map: the mapper iteration on a TRAINED map — the map tools/slam_demo.py builds on the 240-frame synthetic
    sequence (>= 1 500 Adam steps, keyframe growth, pruning: ~209 k Gaussians of which 80-97 % are visible per view, D = 1.2-1.4 M duplicates, tile
    lists of 390 mean / 870 max — the mapper's real workload [REF mp_Mapper.py:200-223], 5x the duplicates of the untrained S-map surfels of the
    headline) —, one hipGraph replay per iteration cycling `n_views` of the run's own keyframe poses (targets: render of a perturbed copy from each pose, so
    gradients are non-zero).  The map is built once per box (`cache`, ~30 s: 240 ray-cast frames + the loop) by a child process.  Reports ms per
    iteration, the kernels' hipEvent times, D / P_vis / longest list per view and the SURVEY 8(d) roofline entry of R7 at that D."""
    import subprocess
    import torch
    from gs_icp_slam_amd import _lib, synth
    from gs_icp_slam_amd.graph import MapperIterationGraph
    from gs_icp_slam_amd.optim import FusedAdam
    from diff_gaussian_rasterization import GaussianRasterizationSettings, GaussianRasterizer
    cache = cache or os.environ.get("GSICP_TRAINED_MAP", "/tmp/gsicp_trained_map.npz")
    t_build = 0.0
    if not os.path.exists(cache):
        t0 = time.perf_counter()
        tmp = cache + f".{os.getpid()}.npz"
        subprocess.run([sys.executable, os.path.join(ROOT, "tools", "slam_demo.py"), "240", "--iters", "6", "--post-iters", "200", "--no-asserts", "--save-map", tmp],
                       check=True, cwd=ROOT, stdout=subprocess.DEVNULL, timeout=900, env=dict(os.environ, GSICP_BENCH_CHILD="1"))
        os.replace(tmp, cache)
        t_build = time.perf_counter() - t0
    z = np.load(cache)
    g = {k: np.ascontiguousarray(z[k]) for k in ("means3D", "shs", "opacities", "scales", "rotations")}
    P = g["means3D"].shape[0]
    poses = z["keyframe_poses"]
    cfg = synth.REPLICA
    W, H = cfg["W"], cfg["H"]
    pick = sorted({int(round(i * (len(poses) - 1) / max(1, n_views - 1))) for i in range(n_views)})
    raw = {"means3D": torch.from_numpy(g["means3D"]), "scales": torch.log(torch.from_numpy(g["scales"])), "rotations": torch.from_numpy(g["rotations"]),
           "opacities": torch.logit(torch.from_numpy(g["opacities"]).clamp(1e-6, 1 - 1e-6)), "shs": torch.from_numpy(g["shs"])}
    params = {k: v.to(dev).contiguous().requires_grad_(True) for k, v in raw.items()}
    rng = np.random.default_rng(5)
    with torch.no_grad():     # targets: the same map with colours and positions nudged (gradients of a map that is still learning)
        t2 = {"means3D": params["means3D"] + torch.from_numpy(rng.normal(0, 2e-3, (P, 3)).astype(np.float32)).to(dev),
              "shs": params["shs"] + torch.from_numpy(rng.normal(0, 0.05, tuple(params["shs"].shape)).astype(np.float32)).to(dev),
              "opacities": torch.from_numpy(g["opacities"]).to(dev), "scales": torch.from_numpy(g["scales"]).to(dev), "rotations": params["rotations"].detach()}
    lib = _lib.load()
    import ctypes
    views = []
    for k in pick:
        cam = synth.make_camera(W, H, cfg["fx"], cfg["fy"], poses[k])
        rs = GaussianRasterizationSettings(image_height=H, image_width=W, tanfovx=cam["tanfovx"], tanfovy=cam["tanfovy"], bg=torch.zeros(3, device=dev),
                                           scale_modifier=1.0, viewmatrix=torch.from_numpy(cam["viewmatrix"]).to(dev), projmatrix=torch.from_numpy(cam["projmatrix"]).to(dev),
                                           sh_degree=0, campos=torch.from_numpy(cam["campos"]).to(dev), prefiltered=False, debug=False)
        with torch.no_grad():
            gd, gc, _, _ = GaussianRasterizer(rs)(means3D=t2["means3D"], means2D=torch.zeros_like(t2["means3D"]), shs=t2["shs"], opacities=t2["opacities"],
                                                  scales=t2["scales"], rotations=t2["rotations"])
        # D, P_vis and the tile lists of the map itself from this pose (the product's own ranges, read from the forward's image scratch)
        m3 = params["means3D"].detach().requires_grad_(True)
        d_, c_, radii, _u = GaussianRasterizer(rs)(means3D=m3, means2D=torch.zeros_like(m3), shs=params["shs"].detach(), opacities=t2["opacities"],
                                                   scales=t2["scales"], rotations=t2["rotations"])
        saved = c_.grad_fn.saved_tensors
        img = saved[9]
        lay = (ctypes.c_size_t * 12)()
        n_dup = int(c_.grad_fn.num_rendered)
        lib.gsicp_raster_layout(P, n_dup, W, H, lay)
        T = ((W + 15) // 16) * ((H + 15) // 16)
        ranges = img[lay[6]: lay[6] + T * 8].cpu().numpy().view(np.uint32).reshape(T, 2).astype(np.int64)
        ln = ranges[:, 1] - ranges[:, 0]
        views.append(dict(rs=rs, gt_color=gc.clone(), gt_depth=gd.clone(), keyframe=int(k), duplicates=n_dup, visible=int((radii > 0).sum()),
                          longest_list=int(ln.max()), mean_list=round(float(ln.mean()), 1)))
        del d_, c_, m3, saved, img
    capacity = int(1.5 * max(v["duplicates"] for v in views)) + 4096
    opt = FusedAdam([{"params": [params[k]], "lr": lr} for k, lr in LRS.items()], lr=0.0, eps=1e-15, capturable=True)
    cam0 = synth.make_camera(W, H, cfg["fx"], cfg["fy"], poses[pick[0]])
    mg = MapperIterationGraph(params, opt, H, W, cam0["tanfovx"], cam0["tanfovy"], sh_degree=0, capacity=capacity, lambda_dssim=0.2, warmup=2)
    v0 = views[0]
    mg.set_view(v0["rs"].viewmatrix, v0["rs"].projmatrix, v0["rs"].campos, v0["gt_color"], v0["gt_depth"])
    mg.capture()
    it = [0]

    def iteration():
        v = views[it[0] % len(views)]
        it[0] += 1
        mg.set_view(v["rs"].viewmatrix, v["rs"].projmatrix, v["rs"].campos, v["gt_color"], v["gt_depth"])
        mg.step()
    for _ in range(2 * len(views)):
        iteration()
    ts = []
    for _ in range(reps):
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        for _ in range(steps):
            iteration()
        torch.cuda.synchronize()
        ts.append((time.perf_counter() - t0) / steps)
    if mg.overflowed() or mg.skipped_steps() > 0:
        raise RuntimeError("trained-map leg: duplicate-list capacity overflowed")
    # per-kernel hipEvent times: the same kernels launched eagerly (one bracket per kernel), over the same view cycle
    rasts = [GaussianRasterizer(v["rs"]._replace(capacity=capacity, raw_params=True)) for v in views]
    opt_e = FusedAdam([{"params": [params[k]], "lr": lr} for k, lr in LRS.items()], lr=0.0, eps=1e-15)
    from gs_icp_slam_amd.loss import mapper_loss_and_grads

    def eager(i):
        v, r = views[i % len(views)], rasts[i % len(views)]
        m2 = torch.zeros_like(params["means3D"], requires_grad=True)
        depth, color, _r, _u2 = r(means3D=params["means3D"], means2D=m2, shs=params["shs"], opacities=params["opacities"], scales=params["scales"],
                                  rotations=params["rotations"])
        parts, gc_, gd_ = mapper_loss_and_grads(color, depth, v["gt_color"], v["gt_depth"], lambda_dssim=0.2)
        torch.autograd.backward((color, depth), (gc_, gd_))
        opt_e.step()
        opt_e.zero_grad(set_to_none=True)
    _lib.profile_enable(True)
    eager(0)
    torch.cuda.synchronize()
    _lib.profile_read()
    n_e = 2 * len(views)
    for i in range(n_e):
        eager(i)
    torch.cuda.synchronize()
    stage = {k: round(1e3 * ms / n_e, 2) for k, (ms, c) in _lib.profile_read().items() if c > 0 and not k.startswith("gicp")}
    _lib.profile_enable(False)
    D = sum(v["duplicates"] for v in views) / len(views)
    Pv = sum(v["visible"] for v in views) / len(views)
    b_r7 = 44.0 * D + 40.0 * W * H + 44.0 * Pv
    us_r7 = stage.get("blend_backward", float("nan"))
    ach = b_r7 / (us_r7 * 1e-6) / 1e9
    ms_it = statistics.median(ts) * 1e3
    mg.release()
    return {"ms_per_iteration": round(ms_it, 4), "iterations_per_s": round(1e3 / ms_it, 1), "block_ms": [round(1e3 * t, 4) for t in ts],
            "gaussians": P, "keyframe_poses_in_the_map": int(len(poses)), "mapper_iterations_that_trained_it": int(z["mapper_iterations"]),
            "views": [{k: v[k] for k in ("keyframe", "duplicates", "visible", "longest_list", "mean_list")} for v in views],
            "duplicates_mean": int(D), "visible_mean": int(Pv), "stage_us": stage, "map_build_s": round(t_build, 1),
            "roofline_trained": {"bound": "hbm", "kernel": "blend_backward_tile_kernel (R7)", "kernel_us": us_r7, "algorithmic_bytes": int(b_r7),
                                 "byte_model": "SURVEY 8(d): 44 D + 40 W H + 44 P_vis", "achieved": round(ach, 2), "peak": HBM_PEAK_GBS, "unit": "GB/s",
                                 "frac": round(ach / HBM_PEAK_GBS, 5)},
            "what": "one hipGraph replay per iteration on the map tools/slam_demo.py trains (240 frames, 6 iterations per frame + 200), cycling keyframe poses of that run; "
                    "stage_us = hipEvent brackets in eager iterations over the same cycle"}


def tracker_vs_map_leg(sizes=(8280, 100_000, 1_000_000), frames=60, fid=155, back=1):
    """The tracker in its STEADY-STATE configuration [REF mp_Tracker.py:282-288; scene/gaussian_model.py:207-215]: the target is the map's
    trackable Gaussians (K of them, out of 2K rows: half fail the opacity / trackable selection), handed over at a tracking keyframe either
    the reference's way — rows selected on the host, `set_input_target(np f32)` + `set_target_covariances_fromqs(np, np)` — or by
    `set_target_from_gaussians` on the device; then 8 280-point frames are aligned against it.  Per K: wall ms of each hand-off (the index
    build is lazy, so the first `align` after a hand-off carries it: `first_align_ms`), steady-state host wall us of `align` and
    `get_source_correspondence`, per-stage device us (hipEvent), LM iterations, the search structure's sizes, and how full its cells are.
    The map's quaternions / scales come from the HIP tracker's own k-NN export of each keyframe (the oracle is not used here)."""
    import torch
    import pygicp
    from gs_icp_slam_amd import _lib, synth
    cfg = synth.REPLICA
    kreg = pygicp.FastGICP()
    kreg.set_max_knn_distance(99999.0)

    def cov_fn(pw):
        kreg.set_input_target(pw)
        kreg.calculate_target_covariance_with_filter()
        return kreg.get_target_rotationsq(), kreg.get_target_scales()

    poses = synth.trajectory(fid + 1)
    src, _, trackable, _ = synth.frame_points(cfg, poses[fid])
    f_src = np.zeros(len(src), np.int32)
    f_src[trackable] = np.arange(1, len(trackable) + 1)
    init = poses[fid - back]
    pc = time.perf_counter
    out = {"source_points": int(len(trackable)), "gate_m": cfg["max_corr"], "initial_guess": f"pose {back} frame(s) earlier "
           f"({1e3 * np.linalg.norm(init[:3, 3] - poses[fid][:3, 3]):.1f} mm away)", "sizes": {}}
    for K in sizes:
        m = synth.tracker_map(K, cov_fn, n_keyframes=(2 if K < 20_000 else 32))
        keep = m["trackable"] & (m["opacity"] > m["opacity_th"])
        tp, tr, ts = (np.ascontiguousarray(m[k][keep]) for k in ("points", "rotations", "scales"))
        reg = pygicp.FastGICP()
        reg.set_max_correspondence_distance(cfg["max_corr"])
        reg.set_max_knn_distance(99999.0)

        def frame(timed=None):
            t0 = pc(); reg.set_input_source(src); reg.set_source_filter(len(trackable), f_src)
            t1 = pc(); T = reg.align(init)
            t2 = pc(); idx, d2 = reg.get_source_correspondence()
            t3 = pc()
            if timed is not None:
                timed.append((t1 - t0, t2 - t1, t3 - t2))
            return T, idx, d2

        # -- the reference's hand-off (host arrays), three times: the first carries allocations
        host = []
        for _ in range(3):
            t0 = pc(); reg.set_input_target(tp)
            t1 = pc(); reg.set_target_covariances_fromqs(tr.reshape(-1), ts.reshape(-1))
            t2 = pc(); frame()
            t3 = pc()
            host.append((t1 - t0, t2 - t1, t3 - t2))
        T_host, idx_host, d2_host = frame()
        # -- the device hand-off
        dev = "cuda"
        g_dev = [torch.from_numpy(m[k]).to(dev) for k in ("points", "rotations", "scales", "opacity")]
        mask_dev = torch.from_numpy(m["trackable"]).to(dev)
        torch.cuda.synchronize()
        devt = []
        for _ in range(3):
            t0 = pc(); n_sel = reg.set_target_from_gaussians(*g_dev, trackable_mask=mask_dev, opacity_th=m["opacity_th"])
            t1 = pc(); frame()
            t2 = pc()
            devt.append((t1 - t0, t2 - t1))
        T_dev, idx_dev, d2_dev = frame()
        # -- steady state
        for _ in range(5):
            frame()
        timed = []
        for _ in range(frames):
            frame(timed)
        st = reg.last_align_stats()
        _lib.profile_enable(True)
        _lib.profile_read()
        for _ in range(20):
            frame()
        stage = {k: round(1e3 * ms / 20, 2) for k, (ms, c) in _lib.profile_read().items() if c > 0 and k.startswith("gicp")}
        _lib.profile_enable(False)
        ix = reg.target_index_stats()
        for lv in ix["levels"]:      # how full the cells are (numpy recount on the host; the library reports the sizes)
            fine = np.floor(tp.astype(np.float64) / (0.5 * lv["cell_m"])).astype(np.int64)
            cc, fc = (np.unique(a_, axis=0, return_counts=True)[1] for a_ in (fine >> 1, fine))
            lv.update(points_per_coarse_cell_mean_max=[round(float(cc.mean()), 2), int(cc.max())],
                      points_per_fine_cell_mean_max=[round(float(fc.mean()), 2), int(fc.max())])
        gt = poses[fid]
        med = lambda i, rows: float(statistics.median(r[i] for r in rows))   # noqa: E731
        out["sizes"][str(K)] = {
            "target_gaussians": int(keep.sum()), "map_rows": int(len(keep)),
            "host_handoff_ms": {"set_input_target": round(1e3 * med(0, host[1:]), 3), "set_target_covariances_fromqs": round(1e3 * med(1, host[1:]), 3),
                                "first_frame_after_it (index build inside align)": round(1e3 * med(2, host[1:]), 3)},
            "device_handoff_ms": {"set_target_from_gaussians": round(1e3 * med(0, devt[1:]), 3), "first_frame_after_it": round(1e3 * med(1, devt[1:]), 3)},
            "frame_us": {"set_input_source+filter": round(1e6 * med(0, timed), 1), "align": round(1e6 * med(1, timed), 1),
                         "get_source_correspondence": round(1e6 * med(2, timed), 1), "frame": round(1e6 * statistics.median(sum(r) for r in timed), 1)},
            "stage_us": stage, "lm_iterations": st["iterations"], "converged": st["converged"],
            "pose_error_mm": round(1e3 * float(np.linalg.norm(np.asarray(T_host, np.float64)[:3, 3] - gt[:3, 3])), 4),
            "in_gate_fraction": round(float((idx_host >= 0).mean()), 4),
            "device_route_equals_host_route": bool(np.array_equal(idx_host, idx_dev) and np.array_equal(d2_host, d2_dev) and np.array_equal(T_host, T_dev)),
            "index": ix,
        }
        del reg, g_dev, mask_dev
    return out


def compact_line(full, legs_path):
    """The contract line: the driver's keys, `roofline` / `roofline_longest_kernel` / `cpu_baseline` without prose, and a flat handful of scalars.  Everything else
    (legs, notes, per-block spreads, per-view arrays) is in the legs file.  tests/test_bench_cli.py holds this under 6 000 characters on a worst-case record."""
    def cut(v, n):
        return v if not isinstance(v, str) or len(v) <= n else v[: n - 3] + "..."

    def pick(d, keys, n=160):
        return None if not d else {k: cut(d.get(k), n) for k in keys if k in d}
    legs = full.get("legs") or {}
    cfg = full.get("config") or {}
    leg = lambda name, key: (legs.get(name) or {}).get(key)   # noqa: E731
    tm = legs.get("mapper_trained_map") or {}
    tm_stage = tm.get("stage_us") or {}
    line = {k: full.get(k) for k in ("metric", "value", "unit", "n_gpus", "steps", "warmup", "ms_per_step", "higher_is_better", "scaling", "vs_baseline", "dtype", "data")}
    line["metric"] = cut(line["metric"], 200)
    line["config"] = {"workload": cut(cfg.get("workload_short") or cfg.get("workload"), 300)}
    line["config"].update({k: cut(cfg.get(k), 200) for k in ("gaussians", "width", "height", "duplicates_per_rank", "visible_gaussians", "keyframe_views", "tracker_workload",
                                                             "lm_iterations", "tracker_target_gaussians", "mapper_iteration", "mp_mode", "parallelism", "world_size", "backend", "cu_split")
                           if cfg.get(k) is not None})
    if cfg.get("mp_bands"):
        line["config"]["mp_bands"] = cfg["mp_bands"].get("mode")
    line["roofline"] = pick(full.get("roofline"), ("bound", "kernel", "kernel_us", "algorithmic_bytes", "achieved", "peak", "unit", "frac", "traffic", "traffic_over_algorithmic",
                                                   "traffic_last_capture"))
    if full.get("roofline"):
        for sub in ("whole_forward", "whole_backward"):
            line["roofline"][sub + "_frac"] = (full["roofline"].get(sub) or {}).get("frac")
    line["roofline_longest_kernel"] = pick(full.get("roofline_longest_kernel"), ("bound", "kernel", "kernel_us", "grid_wide_phases", "us_per_phase", "lm_iterations",
                                                                                "algorithmic_bytes", "achieved", "peak", "unit", "frac", "traffic"), 80)
    line["cpu_baseline"] = pick(full.get("cpu_baseline"), ("value", "unit", "cores", "host_cores", "kind", "sample", "pose_agrees_with_gpu"), 260)
    line.update({
        "block_ms_per_step_p10_p50_p90": full.get("block_ms_per_step_p10_p50_p90"), "repeats": full.get("repeats"), "timed_seconds": full.get("timed_seconds"),
        "render_bwd_ms_per_iter": full.get("render_bwd_ms_per_iter"), "loss_adam_ms_per_iter": full.get("loss_adam_ms_per_iter"),
        "render_bwd_ms_per_iter_trained_map": (round(sum(v for k, v in tm_stage.items() if not k.startswith(("loss_", "adam"))) / 1e3, 4) if tm_stage else None),
        "mapper_iteration_ms_trained_map": tm.get("ms_per_iteration"), "trained_map_duplicates": tm.get("duplicates_mean"),
        "trained_map_r7_frac": (tm.get("roofline_trained") or {}).get("frac"),
        "mapper_only_ms_per_iter": leg("mapper_only", "ms_per_iteration"), "tracker_only_ms_per_frame": leg("tracker_only_steady", "ms_per_frame"),
        "dropin_reference_loop_ms_per_iter": leg("dropin_reference_loop", "ms_per_iteration"),
        "tracker_align_kernel_us": full.get("tracker_align_kernel_us"), "pose_error_deg_mm": full.get("pose_error_deg_mm"),
        "tracker_pose_is_the_true_motion": full.get("tracker_pose_is_the_true_motion"),
        "system_fps": full.get("system_fps"), "ate_cm": full.get("ate_cm"), "psnr": full.get("psnr"), "system_frames": leg("reference_system_run", "frames"),
        "ate_cm_noisy": full.get("ate_cm_noisy"), "ate_cm_noisy_fused": full.get("ate_cm_noisy_fused"),
        "fused_policy": full.get("fused_policy"),
        "step_tum_ms": leg("step_tum", "ms_per_step"),
        "stage_us_per_step": {k: round(v, 1) for k, v in (full.get("stage_us_per_step") or {}).items()},
    })
    for name in ("keyframe_parallel", "tile_sharded"):       # N > 1: the other multi-GPU mode, as two scalars
        if legs.get(name):
            line[name + "_value"] = legs[name].get("value")
            line[name + "_ms_per_step"] = legs[name].get("ms_per_step")
    line["section_wall_s"] = (full.get("section_wall_s") or {}).get("total")
    line["legs_file"] = legs_path
    return line


def _spawn_ranks(n):
    import socket
    import subprocess
    with socket.socket(socket.AF_INET, socket.SOCK_STREAM) as sk:
        sk.bind(("127.0.0.1", 0))
        port = sk.getsockname()[1]
    env = dict(os.environ)
    env.setdefault("HSA_ENABLE_IPC_MODE_LEGACY", "0")      # dmabuf IPC only on this driver: RCCL needs it
    env.setdefault("OMP_NUM_THREADS", "1")
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", f"--nproc-per-node={n}", "--master-addr", "127.0.0.1",
           "--master-port", str(port), os.path.abspath(__file__)] + sys.argv[1:]
    return subprocess.call(cmd, env=env)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=100)
    ap.add_argument("--warmup", type=int, default=10)
    ap.add_argument("--repeats", type=int, default=5, help="minimum number of timed blocks of --steps steps (more are run until --min-seconds); the mean block is reported")
    ap.add_argument("--gaussians", type=int, default=300_000)
    ap.add_argument("--res", choices=["replica", "tum"], default="replica")
    ap.add_argument("--pair", choices=["survey", "basin"], default="survey",
                    help="tracker pair of the headline step: SURVEY 8(d)'s pair verbatim, or the in-basin pair (the other one is timed as a leg)")
    ap.add_argument("--min-seconds", type=float, default=1.0, help="keep adding timed blocks (beyond --repeats) until the timed region is at least this long")
    ap.add_argument("--views", type=int, default=8, help="keyframe views the mapper cycles through (each with its own target images)")
    ap.add_argument("--tracker", choices=["steady", "pair"], default="steady",
                    help="tracker half of the headline step: `steady` = the steady-state configuration (frames of a trajectory against the MAP's trackable "
                         "Gaussians, keyframe cadence inside the timed region); `pair` = rounds 1-3's headline (one S-pair re-aligned against a frame-sized target; --pair)")
    ap.add_argument("--mapper-inflight", type=int, default=2, help="mapper iterations the host may have in flight (queued graph launches) inside a timed block")
    ap.add_argument("--no-reference-leg", action="store_true", help="skip the run of the reference's own two-process system (System FPS / ATE / PSNR keys)")
    ap.add_argument("--system-legs", action="store_true", help="all four runs of the reference's own two-process system on the drop-ins (400 frames clean + 300 frames "
                    "noisy, each untouched and with SURVEY 8(f)'s rows applied: ~120 s); the default runs ONE 400-frame clean run of the untouched system")
    ap.add_argument("--all-legs", action="store_true", help="every diagnostic leg (lockstep, tracker call profile, both S-pairs, tracker vs map sizes, mapper across "
                    "keyframes, the TUM-shaped child run): minutes; the default runs the core legs only")
    ap.add_argument("--legs-file", default=os.environ.get("GSICP_BENCH_LEGS_FILE", os.path.join(ROOT, "bench_legs.json")),
                    help="where the FULL record (every leg, notes, per-block spreads) is written; the one JSON line on stdout stays under 6 KB and names this file")
    ap.add_argument("--full-line", action="store_true", help="print the full record on stdout instead of the compact contract line (tools; NOT for the driver)")
    ap.add_argument("--no-cpu-baseline", action="store_true")
    ap.add_argument("--no-legs", action="store_true", help="skip the extra legs (tracker-only, mapper-only, eager, drop-in reference loop)")
    ap.add_argument("--cpu-seconds", type=float, default=8.0)
    ap.add_argument("--serial", action="store_true", help="run tracker and mapper back-to-back on one thread (default: concurrently)")
    ap.add_argument("--lockstep", action="store_true", help="join the tracker frame and the mapper iteration after EVERY step (round 1's timing loop) instead of "
                    "letting the two halves run their --steps steps at their own pace inside the timed block")
    ap.add_argument("--no-graph", action="store_true", help="drive the mapper iteration eagerly from Python instead of replaying the captured HIP graph")
    ap.add_argument("--only", choices=["tracker", "mapper", "trained"], default=None, help="diagnostics: run only one half (the JSON line is then NOT the contract metric)")
    ap.add_argument("--cu-split", type=int, default=0, help="EXPERIMENT (round 6): the tracker's stream on this many dedicated compute units "
                    "(hipExtStreamCreateWithCUMask, mask bits 0..N-1: spread evenly over the 8 XCDs) and the mapper's stream on the remaining ones, instead of a "
                    "tracker stream sharing all 256; 0 = off")
    ap.add_argument("--mp-bands", choices=["off", "equal", "balanced"], default="off",
                    help="N > 1, --mp-mode tiles: `off` = super-tiles dealt round-robin + all-gather of the image (rounds 3-4, the rehearsed default); `equal` / "
                         "`balanced` (round 5) = contiguous bands of 32-pixel rows per rank + a halo exchange of 2 x 10 rows (0.4 MB instead of 13.7 MB per rank); "
                         "`balanced` places the boundaries by the duplicates per row, averaged over the keyframe views")
    ap.add_argument("--mp-mode", choices=["tiles", "keyframes"], default="tiles",
                    help="N > 1 GPUs: `tiles` (default) = ONE view per step, its screen tiles sharded over the ranks (same optimiser trajectory as 1 GPU: "
                         "strong scaling); `keyframes` = every rank renders its OWN view, one dense gradient all-reduce, N views per optimiser step "
                         "(SURVEY 8e's throughput alternative: NOT result-parity with the reference's one-view-per-step loop; weak scaling).  With "
                         "`tiles` the keyframes mode is also timed, as legs.keyframe_parallel")
    args = ap.parse_args()
    sect = {}              # wall seconds of every section of this command (goes to the legs file: what the default command spends where)
    t_sect = [time.perf_counter()]

    def lap(name):
        now = time.perf_counter()
        sect[name] = round(sect.get(name, 0.0) + now - t_sect[0], 2)
        t_sect[0] = now

    # `python bench.py --gpus N` with N > 1 and no launcher around it (the contract's plain form): start the N ranks ourselves — one process per
    # GPU under torch.distributed.run on 127.0.0.1 with a free port — and pass their output through (rank 0 prints the one JSON line).  Under
    # torchrun (WORLD_SIZE set) this is skipped and the environment decides.  GSICP_BENCH_BACKEND=gloo runs the N ranks on however many GPUs
    # the box has (functional rehearsal of the N > 1 path on a 1-GPU box).
    if args.gpus > 1 and "WORLD_SIZE" not in os.environ:
        return _spawn_ranks(args.gpus)

    import torch
    import torch.distributed as dist
    if os.environ.get("GSICP_BENCH_SPAWN_PROBE") == "1":
        # launcher rehearsal (tests/test_bench_cli.py, no GPU needed): join a gloo group, report who is there, stop before any device work
        w, r = int(os.environ.get("WORLD_SIZE", "1")), int(os.environ.get("RANK", "0"))
        seen = [(r, os.getpid())]
        if w > 1:
            os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
            dist.init_process_group("gloo", rank=r, world_size=w)
            got = [None] * w
            dist.all_gather_object(got, (r, os.getpid()))
            seen = got
            dist.destroy_process_group()
        if r == 0:
            print(json.dumps({"spawn_probe": True, "n_gpus": w, "requested_gpus": args.gpus, "ranks": [s_[0] for s_ in seen],
                              "distinct_processes": len({s_[1] for s_ in seen}), "steps": args.steps, "warmup": args.warmup}))
        return 0
    from gs_icp_slam_amd import _lib, synth
    from gs_icp_slam_amd.activations import activate
    from gs_icp_slam_amd.loss import mapper_loss_and_grads
    from gs_icp_slam_amd.optim import FusedAdam
    from gs_icp_slam_amd.sharded import KeyframeParallelRasterizer, ShardedGaussianRasterizer
    from diff_gaussian_rasterization import GaussianRasterizationSettings, GaussianRasterizer
    import pygicp

    world = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    local_rank = int(os.environ.get("LOCAL_RANK", "0"))
    # N > 1: the captured iteration carries two RCCL calls.  Whether this stack can capture and replay them across N GPUs is probed in a
    # child process with its own rendezvous and a timeout BEFORE this process joins its group (a capture that hangs must not take the
    # benchmark with it); GSICP_BENCH_RCCL_GRAPH=0 / 1 skips the probe and forces eager / graph.
    rccl_graph_probe = None
    if (world > 1 or os.environ.get("GSICP_BENCH_FORCE_COLLECTIVES") == "1") and not args.no_graph and os.environ.get("GSICP_BENCH_BACKEND", "nccl") == "nccl":
        forced = os.environ.get("GSICP_BENCH_RCCL_GRAPH")
        if forced is not None:
            rccl_graph_probe = {"ok": forced == "1", "how": f"GSICP_BENCH_RCCL_GRAPH={forced}"}
        else:
            import subprocess
            env = dict(os.environ, MASTER_ADDR=os.environ.get("MASTER_ADDR", "127.0.0.1"),
                       MASTER_PORT=str(int(os.environ.get("MASTER_PORT", "29500")) + 23))
            for k in list(env):     # the child rendezvous is a plain env:// one, not torchrun's agent store
                if k.startswith("TORCHELASTIC") or k in ("TORCH_NCCL_ASYNC_ERROR_HANDLING",):
                    env.pop(k)
            t0p = time.perf_counter()
            try:
                pr = subprocess.run([sys.executable, os.path.join(ROOT, "tools", "rccl_graph_probe.py")], env=env, capture_output=True, text=True,
                                    timeout=float(os.environ.get("GSICP_BENCH_PROBE_TIMEOUT", "240")))
                rccl_graph_probe = {"ok": pr.returncode == 0, "how": f"tools/rccl_graph_probe.py rc={pr.returncode}",
                                    "seconds": round(time.perf_counter() - t0p, 1)}
                for line in pr.stdout.splitlines():
                    if line.startswith("{"):
                        rccl_graph_probe.update(json.loads(line))
            except subprocess.TimeoutExpired:
                rccl_graph_probe = {"ok": False, "how": "tools/rccl_graph_probe.py timed out", "seconds": round(time.perf_counter() - t0p, 1)}
    # GSICP_BENCH_BACKEND=gloo lets the N > 1 code path be exercised on a box with fewer GPUs than ranks (functional check only).
    backend = os.environ.get("GSICP_BENCH_BACKEND", "nccl")
    dev_index = local_rank if backend == "nccl" else local_rank % max(torch.cuda.device_count(), 1)
    torch.cuda.set_device(dev_index)
    dev = torch.device("cuda", dev_index)
    # GSICP_BENCH_FORCE_COLLECTIVES=1 (diagnostic, one GPU): join a 1-rank RCCL group and run the N > 1 iteration — movers and both
    # collectives captured in the graph — so that the cost of the exchange machinery without wire time can be measured on a 1-GPU box.
    force_coll = world == 1 and os.environ.get("GSICP_BENCH_FORCE_COLLECTIVES") == "1"
    if force_coll:
        os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
        if "MASTER_PORT" not in os.environ:
            import socket
            with socket.socket(socket.AF_INET, socket.SOCK_STREAM) as sk:
                sk.bind(("127.0.0.1", 0))
                os.environ["MASTER_PORT"] = str(sk.getsockname()[1])
        dist.init_process_group("nccl", rank=0, world_size=1, device_id=dev)
    if world > 1:
        os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
        if backend == "nccl":
            dist.init_process_group("nccl", rank=rank, world_size=world, device_id=dev)
        else:
            dist.init_process_group(backend, rank=rank, world_size=world)

    if args.only == "trained":     # diagnostic: legs.mapper_trained_map alone (what tools/capture_profiles.sh runs under rocprofv3)
        leg = trained_map_leg(dev, steps=args.steps, reps=max(1, min(args.repeats, 3)), n_views=args.views)
        print(json.dumps({"metric": "DIAGNOSTIC: mapper iteration on the trained map (legs.mapper_trained_map)", "value": leg["iterations_per_s"], "unit": "iterations/s",
                          "n_gpus": 1, "steps": args.steps, "warmup": args.warmup, "ms_per_step": leg["ms_per_iteration"], "higher_is_better": True,
                          "dtype": "f32", "data": "synthetic", "legs": {"mapper_trained_map": leg}}))
        return 0
    cu_split = None
    if args.cu_split > 0:
        n_cu = torch.cuda.get_device_properties(dev).multi_processor_count
        os.environ["GSICP_TRACKER_CU_MASK"] = f"0:{args.cu_split}"            # read by gsicp_gicp_create
        h = _lib.load().gsicp_stream_create_cu_mask(args.cu_split, n_cu - args.cu_split)
        if not h:
            raise RuntimeError("--cu-split: " + _lib.last_error())
        torch.cuda.set_stream(torch.cuda.ExternalStream(h, device=dev))         # the mapper half (this thread): every launch and graph replay from here on
        cu_split = {"tracker_cus": args.cu_split, "mapper_cus": n_cu - args.cu_split, "device_cus": n_cu}
    cfg = synth.REPLICA if args.res == "replica" else synth.TUM
    W, H = cfg["W"], cfg["H"]
    P = args.gaussians
    # ---------------- mapper inputs (S-map) ----------------
    cam = synth.make_camera(W, H, cfg["fx"], cfg["fy"], synth.DEFAULT_POSE_A)
    g = synth.s_map(P, seed=2)
    # raw (pre-activation) parameters as GaussianModel keeps them [REF scene/gaussian_model.py:105-125]
    raw = {"means3D": torch.from_numpy(g["means3D"]), "scales": torch.log(torch.from_numpy(g["scales"])),
           "rotations": torch.from_numpy(g["rotations"]),
           "opacities": torch.logit(torch.from_numpy(g["opacities"]).clamp(1e-4, 1 - 1e-4)), "shs": torch.from_numpy(g["shs"])}
    params = {k: v.to(dev).contiguous().requires_grad_(True) for k, v in raw.items()}
    use_graph = not args.no_graph
    if force_coll and not (rccl_graph_probe or {}).get("ok"):
        raise RuntimeError(f"GSICP_BENCH_FORCE_COLLECTIVES: RCCL graph-capture probe failed: {rccl_graph_probe}")
    if world > 1:
        ok = torch.tensor([1.0 if (rccl_graph_probe or {}).get("ok") else 0.0], device=dev)
        dist.all_reduce(ok, op=dist.ReduceOp.MIN)          # every rank must have seen the probe succeed
        use_graph = use_graph and bool(ok.item() == 1.0)
    optimizer = FusedAdam([{"params": [params[k]], "lr": lr} for k, lr in LRS.items()], lr=0.0, eps=1e-15, capturable=use_graph)
    rs = GaussianRasterizationSettings(
        image_height=H, image_width=W, tanfovx=cam["tanfovx"], tanfovy=cam["tanfovy"], bg=torch.zeros(3, device=dev), scale_modifier=1.0,
        viewmatrix=torch.from_numpy(cam["viewmatrix"]).to(dev), projmatrix=torch.from_numpy(cam["projmatrix"]).to(dev), sh_degree=0,
        campos=torch.from_numpy(cam["campos"]).to(dev), prefiltered=False, debug=False)
    # Keyframe views the mapper cycles through [REF mp_Mapper.py:197-206: the newest keyframe first, then random.choice over all of them]: the S-map
    # camera of SURVEY 8(d) plus poses along the synthetic trajectory, each with its own target images (render of the perturbed copy from that pose,
    # so gradients are non-zero — SURVEY.md §8d).  Duplicates D and visible Gaussians P_vis differ from view to view, as they do in a run.
    n_views = max(1, args.views)
    traj_v = synth.trajectory(40 * n_views + 1)
    view_poses = [synth.DEFAULT_POSE_A] + [traj_v[40 * i] for i in range(1, n_views)]
    views = []
    with torch.no_grad():
        g2 = synth.s_map(P, seed=2, perturb_seed=3)
        t2 = {k: torch.from_numpy(g2[k]).to(dev) for k in ("means3D", "scales", "rotations", "opacities", "shs")}
        for pose_v in view_poses:
            cam_v = synth.make_camera(W, H, cfg["fx"], cfg["fy"], pose_v)
            rs_v = rs._replace(viewmatrix=torch.from_numpy(cam_v["viewmatrix"]).to(dev), projmatrix=torch.from_numpy(cam_v["projmatrix"]).to(dev),
                               campos=torch.from_numpy(cam_v["campos"]).to(dev))
            gd_v, gc_v, _, _ = ShardedGaussianRasterizer(rs_v)(means3D=t2["means3D"], means2D=torch.zeros_like(t2["means3D"]), shs=t2["shs"],
                                                                opacities=t2["opacities"], scales=t2["scales"], rotations=t2["rotations"])
            views.append(dict(rs=rs_v, gt_color=gc_v.clone(), gt_depth=gd_v.clone()))
        del t2
    gt_color, gt_depth = views[0]["gt_color"], views[0]["gt_depth"]     # the S-map camera: what the single-view legs use
    # N > 1, band mode (round 5): boundaries of the ranks' bands of super-tile rows — identical on every rank (same inputs, same arithmetic)
    bands = None
    if world > 1 and args.mp_bands != "off":
        from gs_icp_slam_amd.sharded import balanced_bands, equal_bands
        if args.mp_bands == "equal":
            bands = equal_bands(H, world)
        else:
            import ctypes
            lib_ = _lib.load()
            gx_ = (W + 15) // 16
            n_rows = (H + 31) // 32
            load = np.zeros(n_rows)
            with torch.no_grad():
                o_, s__, q_ = activate(params["opacities"].detach(), params["scales"].detach(), params["rotations"].detach())
            for v in views:     # duplicates per tile row from the ranges of an unsharded probe forward of this view
                m3 = params["means3D"].detach().requires_grad_(True)
                d_, c_, _r, _u = GaussianRasterizer(v["rs"])(means3D=m3, means2D=torch.zeros_like(m3), shs=params["shs"].detach(), opacities=o_, scales=s__, rotations=q_)
                lay = (ctypes.c_size_t * 12)()
                lib_.gsicp_raster_layout(P, int(c_.grad_fn.num_rendered), W, H, lay)
                T_ = gx_ * ((H + 15) // 16)
                rng_ = c_.grad_fn.saved_tensors[9][lay[6]: lay[6] + T_ * 8].cpu().numpy().view(np.uint32).reshape(T_, 2).astype(np.int64)
                per_row = (rng_[:, 1] - rng_[:, 0]).reshape(-1, gx_).sum(1)
                load += np.array([per_row[2 * r: 2 * r + 2].sum() for r in range(n_rows)], dtype=np.float64)
                del d_, c_, m3
            bands = balanced_bands(load.tolist(), world, H=H)
    shard_kw = dict(bands=bands) if bands is not None else {}
    rast = ShardedGaussianRasterizer(rs, **shard_kw)
    view_i = [0]

    # ---------------- tracker inputs (S-pairs) ----------------
    noise = args.res == "tum"
    pairs = {"survey": synth.s_pair_survey(cfg, noise=noise), "basin": synth.s_pair(cfg, noise=noise)}
    motions = {"survey": "room centre looking +z, 1 deg about y + 2 cm along x (SURVEY 8d verbatim)",
               "basin": ("corner-facing, 0.2/0.3 deg about x/y + 8 mm x + 3 mm z (inside the 2 cm-gate convergence basin)" if cfg["max_corr"] < 0.025
                         else "corner-facing, 1 deg about y + 2 cm along x")}

    def filt(n, tr):
        f = np.zeros(n, np.int32)
        f[tr] = np.arange(1, len(tr) + 1)
        return f

    class TrackerCase:
        def __init__(self, name, reg):
            self.name, self.reg, self.sp = name, reg, pairs[name]
            sp = self.sp
            self.pw = sp["points_a"].astype(np.float64) @ sp["pose_a"][:3, :3].T + sp["pose_a"][:3, 3]
            self.f_src = filt(len(sp["points_b"]), sp["trackable_b"])
            reg.set_max_correspondence_distance(cfg["max_corr"])
            reg.set_max_knn_distance(99999.0)
            reg.set_input_target(self.pw)
            reg.set_target_filter(len(sp["trackable_a"]), filt(len(self.pw), sp["trackable_a"]))
            reg.calculate_target_covariance_with_filter()

        def step(self):
            r, sp = self.reg, self.sp
            r.set_input_source(sp["points_b"])
            r.set_source_filter(len(sp["trackable_b"]), self.f_src)
            T = r.align(sp["pose_a"])
            idx, d2 = r.get_source_correspondence()
            return T, idx, d2

        def step_timed(self, acc):
            """step() with the host wall time of every call added into `acc` (legs.tracker_call_profile)."""
            r, sp, pc = self.reg, self.sp, time.perf_counter
            t0 = pc(); r.set_input_source(sp["points_b"])
            t1 = pc(); r.set_source_filter(len(sp["trackable_b"]), self.f_src)
            t2 = pc(); T = r.align(sp["pose_a"])
            t3 = pc(); idx, d2 = r.get_source_correspondence()
            t4 = pc()
            for k, v in (("set_input_source", t1 - t0), ("set_source_filter", t2 - t1), ("align", t3 - t2), ("get_source_correspondence", t4 - t3), ("frames", 1.0)):
                acc[k] = acc.get(k, 0.0) + v
            return T, idx, d2

        def pose_error(self, T):
            gt = self.sp["pose_b"]
            dR = np.asarray(T, np.float64)[:3, :3] @ gt[:3, :3].T
            return (float(np.degrees(np.linalg.norm(dR - np.eye(3)) / np.sqrt(2.0))), float(1e3 * np.linalg.norm(np.asarray(T, np.float64)[:3, 3] - gt[:3, 3])))

    class SteadyTracker:
        """The tracker's STEADY-STATE frame [REF mp_Tracker.py:186-320]: consecutive frames of the synthetic trajectory (8 280 points each, initial
        guess = the previous frame's pose, ~7 mm / 0.25 deg away) aligned against the MAP's trackable Gaussians — the S-map rows with opacity >
        trackable_opacity_th that carry the trackable flag (half of them) — with the reference's keyframe cadence inside the loop: every
        `map_kf`-th frame a mapping keyframe (the source covariances are exported: get_source_rotationsq + get_source_scales
        [REF mp_Tracker.py:301-309]), every `track_kf`-th a tracking keyframe (the same export, then the target is replaced by the map's current
        trackable Gaussians [REF mp_Tracker.py:256-289]: on the device through set_target_from_gaussians, or — `host=True`, the oracle —
        set_input_target + set_target_covariances_fromqs with host arrays, the reference's own route)."""
        def __init__(self, reg, host=False, n_frames=16, first=150, map_kf=10, track_kf=40):
            self.reg, self.host, self.map_kf, self.track_kf, self.k = reg, host, map_kf, track_kf, 0
            poses = synth.trajectory(first + n_frames + 1)
            self.frames = []
            for j in range(n_frames):
                pts, _, tr, _ = synth.frame_points(cfg, poses[first + 1 + j], **({"noise_seed": 100 + j, "holes": 0.15} if noise else {}))
                self.frames.append(dict(points=pts, trackable=tr, filt=filt(len(pts), tr), init=poses[first + j], gt=poses[first + 1 + j]))
            rng_t = np.random.default_rng(17)
            self.mask = rng_t.random(P) < 0.5
            self.th = 0.09 if args.res == "tum" else 0.05                      # trackable_opacity_th [REF replica.sh:140; tum.sh:140]
            keep = self.mask & (g["opacities"][:, 0] > self.th)
            self.n_target = int(keep.sum())
            if host:
                self.h = [np.ascontiguousarray(g[k][keep]) for k in ("means3D", "rotations", "scales")]
            else:
                self.d = [torch.from_numpy(np.ascontiguousarray(g[k])).to(dev) for k in ("means3D", "rotations", "scales", "opacities")]
                self.dmask = torch.from_numpy(self.mask).to(dev)
            reg.set_max_correspondence_distance(cfg["max_corr"])
            reg.set_max_knn_distance(99999.0)
            self.refresh_target()
            self.worst = [0.0, 0.0]
            self.sp = dict(points_b=self.frames[0]["points"])

        def refresh_target(self):
            if self.host:
                self.reg.set_input_target(self.h[0])
                self.reg.set_target_covariances_fromqs(self.h[1].reshape(-1), self.h[2].reshape(-1))
            else:
                n = self.reg.set_target_from_gaussians(self.d[0], self.d[1], self.d[2], self.d[3], trackable_mask=self.dmask, opacity_th=self.th)
                assert n == self.n_target

        def step(self, acc=None):
            r, pc = self.reg, time.perf_counter
            k = self.k
            self.k += 1
            f = self.frames[k % len(self.frames)]
            t0 = pc(); r.set_input_source(f["points"])
            t1 = pc(); r.set_source_filter(len(f["trackable"]), f["filt"])
            t2 = pc(); T = r.align(f["init"])
            t3 = pc(); idx, d2 = r.get_source_correspondence()
            t4 = pc()
            if k % self.map_kf == 0 or k % self.track_kf == 0:
                r.get_source_rotationsq(); r.get_source_scales()
            if k % self.track_kf == 0 and k > 0:
                self.refresh_target()
            t5 = pc()
            if acc is not None:
                for name, v in (("set_input_source", t1 - t0), ("set_source_filter", t2 - t1), ("align", t3 - t2), ("get_source_correspondence", t4 - t3),
                                ("keyframe_work", t5 - t4), ("frames", 1.0)):
                    acc[name] = acc.get(name, 0.0) + v
            e = self.pose_error(T, f["gt"])
            self.worst = [max(self.worst[0], e[0]), max(self.worst[1], e[1])]
            self.last_gt = f["gt"]
            return T, idx, d2

        def step_timed(self, acc):
            return self.step(acc)

        def pose_error(self, T, gt=None):
            gt = self.last_gt if gt is None else gt
            dR = np.asarray(T, np.float64)[:3, :3] @ gt[:3, :3].T
            return (float(np.degrees(np.linalg.norm(dR - np.eye(3)) / np.sqrt(2.0))), float(1e3 * np.linalg.norm(np.asarray(T, np.float64)[:3, 3] - gt[:3, 3])))

    steady = args.tracker == "steady"
    trk = SteadyTracker(pygicp.FastGICP()) if steady else TrackerCase(args.pair, pygicp.FastGICP())
    last = {}

    # The reference runs the tracker and the mapper as two concurrent processes on one GPU [REF gs_icp_slam.py:121-131].
    # Here: the tracker frame runs on a worker thread (its C calls release the GIL and use the tracker's own HIP stream)
    # while the main thread drives the mapper iteration on torch's stream; a step ends when both are done.
    import queue
    import threading
    jobs, done = queue.Queue(), queue.Queue()

    def tracker_worker():
        torch.cuda.set_device(dev_index)
        while True:
            job = jobs.get()
            if job is None:
                return
            case, n = (job if isinstance(job, tuple) and not isinstance(job[0], int) else (trk, job))
            r = None
            if isinstance(n, tuple):         # (frames, accumulator): the timed variant of the frame (legs.tracker_call_profile)
                for _ in range(n[0]):
                    r = case.step_timed(n[1])
                done.put(r)
                continue
            for _ in range(n):
                r = case.step()
            done.put(r)
    worker = None
    if not args.serial and args.only is None:
        worker = threading.Thread(target=tracker_worker, daemon=True)
        worker.start()

    def activated(p=params):   # GaussianModel.get_opacity / get_scaling / get_rotation [REF scene/gaussian_model.py:105-125], one fused launch
        o, s_, q = activate(p["opacities"], p["scales"], p["rotations"])
        return dict(means3D=p["means3D"], shs=p["shs"], opacities=o, scales=s_, rotations=q)

    def eager_iteration():
        """One iteration of Mapper.mapping [REF mp_Mapper.py:219-248] with the fused operators, launched from Python, on the next keyframe view."""
        vi = view_i[0] % n_views
        view_i[0] += 1
        rast, v = rasts[vi], views[vi]
        a = activated()
        means2D = torch.zeros_like(a["means3D"], requires_grad=True)
        depth, color, radii, used = rast(means3D=a["means3D"], means2D=means2D, shs=a["shs"], opacities=a["opacities"],
                                         scales=a["scales"], rotations=a["rotations"])
        shard = rast.loss_shard()        # N > 1: the loss is sharded with the tiles (this rank's 32x32 blocks)
        parts, g_color, g_depth = mapper_loss_and_grads(color, depth, v["gt_color"], v["gt_depth"], lambda_dssim=0.2, tile_mod=shard[0], tile_rem=shard[1])
        if shard[0] > 1:
            rast.attach_loss_share(parts)
        torch.autograd.backward((color, depth), (g_color, g_depth))
        optimizer.step()
        optimizer.zero_grad(set_to_none=True)
        return parts[0], radii

    # Duplicate-list capacity for the sync-free forward: 1.5x the count of one probe forward (per rank: each rank bins its own tiles).
    def probe_capacity():
        cap = max(8 * P // world, 1 << 20)
        worst_r, worst_vis = 0, 0
        for v in views:
            while True:   # plain rasteriser on this rank's tiles: no collective inside a loop whose trip count may differ between ranks
                own = rast.raster_settings if bands is not None else None       # band mode: this rank's band code
                probe = GaussianRasterizer(v["rs"]._replace(capacity=cap, tile_mod=(own.tile_mod if own else world), tile_rem=(own.tile_rem if own else rank)))
                with torch.no_grad():
                    a0 = activated()
                    radii_p = probe(means3D=a0["means3D"], means2D=torch.zeros_like(a0["means3D"]), shs=a0["shs"], opacities=a0["opacities"],
                                    scales=a0["scales"], rotations=a0["rotations"])[2]
                r = int(probe.num_rendered.item())
                if r <= cap:
                    break
                cap *= 2
            v["duplicates"], v["visible"] = r, int((radii_p > 0).sum())
            worst_r, worst_vis = max(worst_r, r), max(worst_vis, v["visible"])
        return int(1.5 * worst_r) + 4096, int(1.5 * worst_vis) + 1024
    capacity, vis_capacity = probe_capacity()      # over ALL views; vis_capacity: rows of the static gradient all-reduce block (same on every rank: radii are replicated)
    rasts = [ShardedGaussianRasterizer(v["rs"]._replace(capacity=capacity), **shard_kw) for v in views]   # eager iterations also run without the forward's host sync
    rast = rasts[0]

    mg = None
    capture_error = None
    mapper_iteration = eager_iteration
    if use_graph:
        # Single GPU: the whole iteration is one hipGraph launch (gs_icp_slam_amd/graph.py); the keyframe (camera + targets) is
        # re-selected before every replay, as the reference's mapper does [REF mp_Mapper.py:205-217].
        from gs_icp_slam_amd.graph import MapperIterationGraph
        # N > 1: the tile-sharded rasteriser with its static-size exchange (tile chunks all-gathered, visible gradient rows all-reduced) is
        # captured in the same graph, RCCL calls included (gs_icp_slam_amd/sharded.py)
        factory = (lambda rs_: ShardedGaussianRasterizer(rs_, vis_capacity=vis_capacity, force_collectives=force_coll, **shard_kw)) if (world > 1 or force_coll) else None
        mg = MapperIterationGraph(params, optimizer, H, W, cam["tanfovx"], cam["tanfovy"], sh_degree=0, capacity=capacity,
                                  lambda_dssim=0.2, warmup=2, rasterizer_factory=factory)
        mg.set_view(rs.viewmatrix, rs.projmatrix, rs.campos, gt_color, gt_depth)
        # A capture that FAILS (round 5's took the whole process down from the process group's watchdog thread; graph.py now captures
        # thread-locally behind a drained watchdog) must cost the graph, not the benchmark line: every rank falls back to the eager iteration together.
        capture_error = None
        try:
            if os.environ.get("GSICP_BENCH_FAIL_CAPTURE") == "1":      # test hook (tests/test_bench_gpu.py): the fallback below, without a real failure
                raise RuntimeError("GSICP_BENCH_FAIL_CAPTURE=1")
            mg.capture()
        except Exception as e:   # noqa: BLE001
            capture_error = f"{type(e).__name__}: {e}"[:160]
        if world > 1:
            okc = torch.tensor([0.0 if capture_error else 1.0], device=dev)
            dist.all_reduce(okc, op=dist.ReduceOp.MIN)
            if okc.item() != 1.0 and capture_error is None:
                capture_error = "another rank's capture failed"
        if capture_error is not None:
            try:
                mg.release()
            except Exception:   # noqa: BLE001
                pass
            mg = None
            torch.cuda.synchronize()
        else:
            def mapper_iteration():   # noqa: F811
                v = views[view_i[0] % n_views]
                view_i[0] += 1
                mg.set_view(v["rs"].viewmatrix, v["rs"].projmatrix, v["rs"].campos, v["gt_color"], v["gt_depth"])
                return mg.step(), mg.radii

    def step():
        if args.only == "tracker":
            T, idx, d2 = trk.step()
            last.update(T=T)
            return
        if args.only == "mapper":
            loss, radii = mapper_iteration()
            last.update(loss=loss, radii=radii)
            return
        if worker is not None:
            jobs.put(1)
            loss, radii = mapper_iteration()
            T, idx, d2 = done.get()
        else:
            T, idx, d2 = trk.step()
            loss, radii = mapper_iteration()
        last.update(T=T, loss=loss, radii=radii)

    def barrier():
        if world > 1:
            dist.barrier()
        torch.cuda.synchronize()

    inflight = [torch.cuda.Event() for _ in range(max(1, args.mapper_inflight))]

    def free_running_block(steps):
        """`steps` tracker frames on the worker thread and `steps` mapper iterations on this one, each half at its own pace, as the
        reference's two processes run [REF gs_icp_slam.py:121-131: Tracker.run and Mapper.run never wait for each other per frame]; the
        block ends when BOTH halves have finished all their steps."""
        jobs.put(steps)
        for i in range(steps):
            # bounded run-ahead, as in the fused in-system loop (gs_icp_slam_amd/refglue.py): a graph launch returns at once, so this thread could queue
            # the whole block ahead of the GPU, and the tracker's tracking keyframe — whose hand-off is ordered after everything queued on the
            # mapper's stream — would wait for all of it (measured: 15 ms stalls, 0.47 instead of 0.36 ms per step at 100-step blocks).  The
            # reference's own mapper is throttled by its synchronous forward; here at most `--mapper-inflight` iterations are in flight.
            ev = inflight[i % len(inflight)]
            if i >= len(inflight):
                ev.synchronize()
            loss, radii = mapper_iteration()
            ev.record()
        T, idx, d2 = done.get()
        last.update(T=T, loss=loss, radii=radii)

    def timed_blocks(fn, steps, repeats, whole=None, min_seconds=0.0):
        out = []
        while True:
            if len(out) >= repeats:      # more blocks until the timed region is long enough; with several ranks rank 0's clock decides for all
                go = sum(out) < min_seconds and len(out) < 2000
                if world > 1:
                    flag = torch.tensor([1.0 if go else 0.0], device=dev)
                    dist.broadcast(flag, 0)
                    go = flag.item() != 0.0
                if not go:
                    break
            barrier()
            t0 = time.perf_counter()
            if whole is not None:
                whole(steps)
            else:
                for _ in range(steps):
                    fn()
            barrier()
            dt = time.perf_counter() - t0
            if world > 1:
                tmax = torch.tensor([dt], dtype=torch.float64, device=dev)
                dist.all_reduce(tmax, op=dist.ReduceOp.MAX)
                dt = float(tmax.item())
            out.append(dt)
        return out

    lap("imports_inputs_capture")
    for _ in range(args.warmup):
        step()
    free_running = worker is not None and not args.lockstep
    blocks = timed_blocks(step, args.steps, max(1, args.repeats), whole=free_running_block if free_running else None, min_seconds=args.min_seconds)
    dt = sum(blocks) / len(blocks)     # every timed step over every timed second: blocks with a tracking keyframe (every 40th frame) count at their share
    if mg is not None and (mg.overflowed() or mg.skipped_steps() > 0):
        raise RuntimeError(f"capacity overflowed during the timed region: R = {int(mg.num_rendered.item())} (capacity {mg.capacity}), "
                           f"{mg.skipped_steps()} optimiser steps skipped")
    if mg is None and int(rast.inner.num_rendered.item()) > capacity:
        raise RuntimeError("duplicate-list capacity overflowed during the timed region")
    align_stats = trk.reg.last_align_stats() if args.only != "mapper" else {}
    lap("warmup_and_timed_region")

    # ---------------- N > 1: the throughput mode, data-parallel over keyframes (SURVEY 8e alternative), timed on ALL ranks ----------------
    # Every rank renders ITS OWN view of the same map (full image, plain single-GPU rasteriser), one dense all-reduce sums the parameter
    # gradients, the replicated optimiser takes one step per N views.  NOT result-parity with the reference's one-view-per-step loop.
    kf_leg = None
    mgk = None
    if (world > 1 or force_coll) and (not args.no_legs or args.mp_mode == "keyframes") and args.only != "tracker":
        from gs_icp_slam_amd.graph import MapperIterationGraph as _KMG
        pose_r = synth.DEFAULT_POSE_A @ synth.se3((0.0, 3.0 * rank, 0.0), (0.03 * rank, 0.0, 0.0))
        cam_r = synth.make_camera(W, H, cfg["fx"], cfg["fy"], pose_r)
        rs_r = rs._replace(viewmatrix=torch.from_numpy(cam_r["viewmatrix"]).to(dev), projmatrix=torch.from_numpy(cam_r["projmatrix"]).to(dev),
                           campos=torch.from_numpy(cam_r["campos"]).to(dev))
        with torch.no_grad():
            g2 = synth.s_map(P, seed=2, perturb_seed=3)
            t2 = {k: torch.from_numpy(g2[k]).to(dev) for k in ("means3D", "scales", "rotations", "opacities", "shs")}
            gtd_r, gtc_r, _, _ = GaussianRasterizer(rs_r)(means3D=t2["means3D"], means2D=torch.zeros_like(t2["means3D"]), shs=t2["shs"],
                                                          opacities=t2["opacities"], scales=t2["scales"], rotations=t2["rotations"])
            gtd_r, gtc_r = gtd_r.clone(), gtc_r.clone()
            del t2
            cap_k = max(8 * P, 1 << 20)
            while True:
                pr = GaussianRasterizer(rs_r._replace(capacity=cap_k))
                a0 = activated()
                pr(means3D=a0["means3D"], means2D=torch.zeros_like(a0["means3D"]), shs=a0["shs"], opacities=a0["opacities"], scales=a0["scales"],
                   rotations=a0["rotations"])
                r_full = int(pr.num_rendered.item())
                if r_full <= cap_k:
                    break
                cap_k *= 2
            cap_k = int(1.5 * r_full) + 4096
        opt_k = FusedAdam([{"params": [params[k]], "lr": lr} for k, lr in LRS.items()], lr=0.0, eps=1e-15, capturable=use_graph)
        if use_graph:
            mgk = _KMG(params, opt_k, H, W, cam_r["tanfovx"], cam_r["tanfovy"], sh_degree=0, capacity=cap_k, lambda_dssim=0.2, warmup=2,
                       rasterizer_factory=lambda rs_: KeyframeParallelRasterizer(rs_, force_collectives=force_coll))
            mgk.set_view(rs_r.viewmatrix, rs_r.projmatrix, rs_r.campos, gtc_r, gtd_r)
            mgk.capture()
            kf_holder = mgk.rasterizer.holder

            def kf_iteration():
                mgk.set_view(rs_r.viewmatrix, rs_r.projmatrix, rs_r.campos, gtc_r, gtd_r)
                return mgk.step(), mgk.radii
        else:
            kf_rast = KeyframeParallelRasterizer(rs_r._replace(capacity=cap_k), force_collectives=force_coll)
            kf_holder = kf_rast.holder

            def kf_iteration():
                a = activated()
                means2D = torch.zeros_like(a["means3D"], requires_grad=True)
                depth, color, radii, used = kf_rast(means3D=a["means3D"], means2D=means2D, shs=a["shs"], opacities=a["opacities"],
                                                    scales=a["scales"], rotations=a["rotations"])
                parts, g_color, g_depth = mapper_loss_and_grads(color, depth, gtc_r, gtd_r, lambda_dssim=0.2)
                torch.autograd.backward((color, depth), (g_color, g_depth))
                opt_k.step()
                opt_k.zero_grad(set_to_none=True)
                return parts[0], radii

        def kf_step():
            if worker is not None and args.only is None:
                jobs.put(1)
                kf_iteration()
                done.get()
            else:
                if args.only is None:
                    trk.step()
                kf_iteration()

        def kf_free_block(steps):
            jobs.put(steps)
            for _ in range(steps):
                kf_iteration()
            done.get()
        for _ in range(max(3, args.warmup // 2)):
            kf_step()
        kf_blocks = timed_blocks(kf_step, args.steps, max(1, args.repeats), whole=kf_free_block if (free_running and args.only is None) else None)
        dtk = sum(kf_blocks) / len(kf_blocks)
        if use_graph and (mgk.overflowed() or mgk.skipped_steps() > 0):
            raise RuntimeError("keyframe-parallel leg: capacity overflowed during the timed region")
        kf_leg = {"mode": "keyframes", "value": round(world * args.steps / dtk, 3), "unit": "frames/s (N tracker-frame replicas + N mapper views per step)",
                  "views_per_step": world, "ms_per_step": round(1e3 * dtk / args.steps, 4), "scaling": "weak",
                  "block_ms_per_step": [round(1e3 * b / args.steps, 4) for b in kf_blocks],
                  "gradient_all_reduce_bytes_per_rank": kf_holder.last_volume_bytes, "duplicates_per_rank": r_full,
                  "mapper_iteration": "one hipGraph replay per iteration (dense gradient all-reduce captured inside)" if use_graph else "eager launches from Python",
                  "what": "data-parallel over keyframes: every rank renders its own view of the replicated map, one dense all-reduce(sum) of the 14 parameter-"
                          "gradient floats per Gaussian + a flag word, replicated Adam step on the N views' summed loss; tracker replicas on every rank; "
                          "NOT result-parity with the reference's one-view-per-step loop [REF mp_Mapper.py:200-206]"}
        if use_graph:
            mgk.release()     # the graph replays RCCL kernels: gone before the communicator is, and its pools are free for the legs below
            mgk = None

    # ---------------- per-kernel hipEvent times ----------------
    # kernels inside a replayed graph carry no HIP events: the SAME kernels on the same inputs are timed (one hipEvent bracket per kernel) in eager iterations right after the
    # timed region, the tracker stages in tracker-only frames (rocprofv3's kernel trace of this command sees all of them and must agree —
    # profiles/README.md)
    _lib.profile_enable(True)
    _lib.profile_read()
    n_e = 20
    per_launch_us = {}
    if args.only != "tracker":
        eager_iteration()
        torch.cuda.synchronize()
        _lib.profile_read()
        for _ in range(n_e):
            eager_iteration()
        torch.cuda.synchronize()
        per_launch_us.update({k: 1e3 * ms / n_e for k, (ms, c) in _lib.profile_read().items() if c > 0 and not k.startswith("gicp")})
    if args.only != "mapper":
        for _ in range(3):
            trk.step()
        _lib.profile_read()
        for _ in range(n_e):
            trk.step()
        per_launch_us.update({k: 1e3 * ms / n_e for k, (ms, c) in _lib.profile_read().items() if c > 0 and k.startswith("gicp")})
    _lib.profile_enable(False)
    lap("per_kernel_hipevent_times")

    # ---------------- D (duplicates), P_vis: per keyframe view (counted by the capacity probe), averaged over the cycle ----------------
    D_views, Pvis_views = [v["duplicates"] for v in views], [v["visible"] for v in views]
    D_local = int(round(sum(D_views) / len(D_views)))
    P_vis = int(round(sum(Pvis_views) / len(Pvis_views)))
    T_tiles = ((W + 15) // 16) * ((H + 15) // 16)

    # ---------------- roofline: SURVEY 8(d) byte model ----------------
    roofline = None
    if args.only != "tracker":
        n_pass = 6
        WHr, Tr = W * H / world, T_tiles / world
        b_r7 = 44.0 * D_local + 40.0 * WHr + 44.0 * P_vis                       # blend backward (R7)
        b_bwd = b_r7 + 184.0 * P                                                # + R8/R9
        b_fwd = 128.0 * P + D_local * (64.0 + 24.0 * n_pass) + 24.0 * WHr + 8.0 * Tr
        fwd_stages = ["preprocess", "emit", "split_hist", "split_colscan", "tile_scan_lpt", "split_scatter", "tile_sort", "blend_forward"]
        bwd_stages = ["blend_backward", "entry_run_sum", "preprocess_backward"]
        us_r7 = per_launch_us.get("blend_backward", float("nan"))
        us_bwd = sum(per_launch_us.get(k, 0.0) for k in bwd_stages)
        us_fwd = sum(per_launch_us.get(k, 0.0) for k in fwd_stages)
        gbs = lambda b, us: b / (us * 1e-6) / 1e9   # noqa: E731
        ach = gbs(b_r7, us_r7)
        # design byte count of the kernel as built: 4 strip waves each read the list word (16 B / duplicate), staged
        # 48-byte records, per-pixel state, 48-byte gradient slot writes per (entry, strip)
        design_bytes = 64.0 * D_local + 40.0 * WHr + 48.0 * D_local
        traffic, traffic_src, note = None, None, ("working set (~60 MB) sits in the 256 MiB Infinity Cache: the HBM fraction is a formality; the kernel runs "
                                                  "~80 % VALU-busy and tracks the per-entry dependent chain (DESIGN 3.3)")
        if world == 1 and args.res == "replica" and P == 300_000:
            for tag in ("r06", "r05", "r04", "r03", "r02", "r01"):   # PMC passes of this command, collected by tools/capture_profiles.sh (counters cannot be read in-process)
                tp = os.path.join(ROOT, "profiles", f"{tag}_pmc_traffic.json")
                if os.path.exists(tp):
                    tj = json.load(open(tp)).get("blend_backward")
                    if tj:
                        traffic, traffic_src = int(tj["fetch_bytes"] + tj["write_bytes"]), f"profiles/{tag}_pmc_traffic.json (rocprofv3 FETCH_SIZE + WRITE_SIZE passes of this command by tools/capture_profiles.sh; PMC counters cannot be read in-process, so this is the LAST CAPTURE, not this run)"
                    sq = os.path.join(ROOT, "profiles", f"{tag}_rocprofv3_pmc_sq.csv")
                    if os.path.exists(sq):
                        import csv
                        for row in csv.DictReader(open(sq)):
                            if row["kernel"].startswith("blend_backward") and float(row.get("SQ_INSTS_VALU", 0) or 0) > 0:
                                valu = float(row["SQ_INSTS_VALU"])
                                note += (f"; SQ_INSTS_VALU = {valu / 1e6:.1f} M wave-instructions x 4 cycles / 1024 SIMDs / 2.4 GHz = "
                                         f"{valu * 4.0 / 1024.0 / 2.4e3:.0f} us issue floor ({os.path.basename(sq)})")
                                break
                    break
        traffic_run, traffic_why = None, "not measured: diagnostic / multi-GPU / child run"
        if rank == 0 and world == 1 and args.only is None and not args.no_legs and os.environ.get("GSICP_BENCH_CHILD") != "1" \
                and os.environ.get("GSICP_BENCH_PMC", "1") != "0":
            pmc, traffic_why = _measure_pmc_traffic("blend_backward_tile_kernel")
            if pmc is not None:
                traffic_run = int(pmc["FETCH_SIZE"] + pmc["WRITE_SIZE"])
                traffic_why = (f"measured in THIS run: two child passes `rocprofv3 --pmc FETCH_SIZE|WRITE_SIZE --kernel-trace -- python bench.py --only mapper "
                               f"--steps 8` (mean over {pmc['FETCH_SIZE_launches']} launches): FETCH_SIZE {int(pmc['FETCH_SIZE'])} B + WRITE_SIZE {int(pmc['WRITE_SIZE'])} B, raw counters; "
                               "calibration on this box's access patterns (profiles/r03_pmc_calibration.json): FETCH_SIZE reads a coalesced 16 B/lane stream at 0.50x and a "
                               "gather of 48-byte records at 1.55x of the bytes requested, WRITE_SIZE 1.00x / 1.28x — this kernel's fetches are ~2/3 record gathers, so "
                               "the true figure lies between 1x and 1.3x of the raw sum")
        roofline = {"bound": "hbm", "kernel": "blend_backward_tile_kernel (R7)", "achieved": round(ach, 2), "peak": HBM_PEAK_GBS, "unit": "GB/s",
                    "frac": round(ach / HBM_PEAK_GBS, 5), "traffic": traffic_run, "traffic_how": traffic_why,
                    "traffic_over_algorithmic": (round(traffic_run / b_r7, 3) if traffic_run else None),
                    "traffic_last_capture": traffic, "traffic_source": traffic_src, "kernel_us": round(us_r7, 2),
                    "algorithmic_bytes": int(b_r7), "byte_model": "SURVEY 8(d): 44 D + 40 W H + 44 P_vis",
                    "design_bytes": int(design_bytes), "design_frac": round(gbs(design_bytes, us_r7) / HBM_PEAK_GBS, 5),
                    "whole_backward": {"algorithmic_bytes": int(b_bwd), "us": round(us_bwd, 2), "frac": round(gbs(b_bwd, us_bwd) / HBM_PEAK_GBS, 5),
                                       "byte_model": "44 D + 40 W H + 44 P_vis + 184 P", "kernels": bwd_stages},
                    "whole_forward": {"algorithmic_bytes": int(b_fwd), "us": round(us_fwd, 2), "frac": round(gbs(b_fwd, us_fwd) / HBM_PEAK_GBS, 5),
                                      "byte_model": "128 P + D (64 + 24 x 6) + 24 W H + 8 T", "kernels": fwd_stages},
                    "note": note}
    roofline_align = None
    if args.only != "mapper" and align_stats:
        us_al = per_launch_us.get("gicp_align")
        m_src = len(trk.sp["points_b"])
        its, trials = align_stats.get("iterations") or 0, align_stats.get("lm_trials") or 0
        phases = trials + 1       # the opening linearisation + one phase per LM trial (an accepted trial carries the next linearisation)
        b_al = 96.0 * m_src * max(its, 1) + 48.0 * m_src
        if us_al:
            roofline_align = {"bound": "hbm", "kernel": "gicp_align_kernel (T3-T6, the LONGEST kernel of the step)", "kernel_us": round(us_al, 2), "grid_wide_phases": phases,
                              "us_per_phase": round(us_al / phases, 2), "lm_iterations": its, "algorithmic_bytes": int(b_al),
                              "byte_model": "SURVEY 8(d): 96 B per trackable source point per outer iteration + 48 B per point once",
                              "achieved": round(b_al / (us_al * 1e-6) / 1e9, 2), "peak": HBM_PEAK_GBS, "unit": "GB/s",
                              "frac": round(b_al / (us_al * 1e-6) / 1e9 / HBM_PEAK_GBS, 6), "traffic": None,
                              "note": "latency-bound by construction (SURVEY 8d: 'report us per align, outer iterations and launches as the primary figures, HBM "
                                      "fraction as a formality'): one persistent launch, every grid-wide phase = NN search + linearisation + wave/LDS reduce + "
                                      "grid barrier + serial 6x6 solve; the actionable figure is us_per_phase"}

    # ---------------- legs (rank 0, single GPU) ----------------
    legs = None
    lap("roofline_and_pmc_passes")
    if rank == 0 and world == 1 and not args.no_legs and args.only is None:
        legs = {}
        reps = max(3, args.repeats)

        def rate(fn, n, warm=3):
            for _ in range(warm):
                fn()
            ts = timed_blocks(fn, n, reps)
            return statistics.median(ts) / n

        # -- the same step with both halves joined after EVERY step (round 1's timing loop; the queue hand-shake per step makes it slower and
        #    bimodal from run to run)
        if worker is not None and free_running and args.all_legs:
            s_lock = rate(step, 100)
            legs["lockstep_step"] = {"frames_per_s": round(1.0 / s_lock, 1), "ms_per_step": round(1e3 * s_lock, 4),
                                     "what": "tracker frame and mapper iteration joined after every step (round-1 loop)"}
        # -- where the tracker's frame goes on the HOST side, alone and next to the free-running mapper: wall time of each of the four calls of a frame
        #    [REF mp_Tracker.py:191-199, 231] (the GPU work of a call is inside it only where the call has to wait: align, get_source_correspondence)
        if worker is not None and free_running and args.all_legs:
            prof = {}
            for mode in ("alone", "co_tenant"):
                acc = {}
                for _ in range(2):
                    acc.clear()
                    torch.cuda.synchronize()
                    jobs.put((200, acc))
                    if mode == "co_tenant":
                        for i_ in range(200):       # same bounded run-ahead as the timed blocks
                            ev_ = inflight[i_ % len(inflight)]
                            if i_ >= len(inflight):
                                ev_.synchronize()
                            mapper_iteration()
                            ev_.record()
                    done.get()
                    torch.cuda.synchronize()
                n_f = acc.pop("frames")
                prof[mode] = {k: round(1e6 * v / n_f, 1) for k, v in acc.items()}
                prof[mode]["frame"] = round(sum(prof[mode].values()), 1)
            legs["tracker_call_profile_us"] = prof
        # -- tracker alone: the steady-state frame and both S-pairs (frame-sized target)
        motions["steady"] = ("consecutive frames of the synthetic trajectory (~7 mm / 0.25 deg apart) against the map's trackable Gaussians; every 10th frame "
                             "exports the source covariances, every 40th replaces the target (set_target_from_gaussians)")
        cases = {("steady" if steady else args.pair): trk}
        for name in (("steady", "survey", "basin") if args.all_legs else ("steady",)):
            if name not in cases:
                cases[name] = SteadyTracker(pygicp.FastGICP()) if name == "steady" else TrackerCase(name, pygicp.FastGICP())
        for name, case in cases.items():
            s_frame = rate(case.step, 100)
            T, idx, d2 = case.step()
            st = case.reg.last_align_stats()
            _lib.profile_enable(True)
            _lib.profile_read()
            for _ in range(20):
                case.step()
            pr = {k: round(1e3 * ms / 20, 2) for k, (ms, c) in _lib.profile_read().items() if c > 0 and k.startswith("gicp")}
            _lib.profile_enable(False)
            ang, mm = tuple(case.worst) if name == "steady" else case.pose_error(T)     # steady: worst over every frame tracked
            legs[f"tracker_only_{name}"] = {"frames_per_s": round(1.0 / s_frame, 1), "ms_per_frame": round(1e3 * s_frame, 4), "motion": motions[name],
                                            "lm_iterations": st["iterations"], "converged": st["converged"], "stage_us": pr,
                                            "pose_error_deg_mm": [round(ang, 4), round(mm, 3)], "correspondence_ratio": round(float((idx >= 0).mean()), 3)}
            if name == "steady":
                legs["tracker_only_steady"].update(target_gaussians=case.n_target, worst_pose_error_deg_mm=[round(case.worst[0], 4), round(case.worst[1], 3)],
                                                   index=case.reg.target_index_stats())
        # -- the tracker against MAP-sized targets (its steady-state configuration after the first tracking keyframe)
        lap("tracker_legs")
        if args.all_legs and os.environ.get("GSICP_BENCH_MAP_LEG", "1") != "0":
            legs["tracker_vs_map"] = tracker_vs_map_leg()
            lap("tracker_vs_map")
        # -- mapper alone: graph replay, eager fused
        s_it = rate(lambda: mapper_iteration(), 100)
        legs["mapper_only"] = {"iterations_per_s": round(1.0 / s_it, 1), "ms_per_iteration": round(1e3 * s_it, 4),
                               "launch": "one hipGraph replay per iteration" if mg is not None else "eager"}
        if mg is not None:   # the same fused operators launched eagerly from Python (what N > 1 runs today)
            opt_e = FusedAdam([{"params": [params[k]], "lr": lr} for k, lr in LRS.items()], lr=0.0, eps=1e-15)
            optimizer_ref = [opt_e]

            def eager_fused():
                a = activated()
                means2D = torch.zeros_like(a["means3D"], requires_grad=True)
                depth, color, radii, used = rast(means3D=a["means3D"], means2D=means2D, shs=a["shs"], opacities=a["opacities"],
                                                 scales=a["scales"], rotations=a["rotations"])
                parts, g_color, g_depth = mapper_loss_and_grads(color, depth, gt_color, gt_depth, lambda_dssim=0.2)
                torch.autograd.backward((color, depth), (g_color, g_depth))
                optimizer_ref[0].step()
                optimizer_ref[0].zero_grad(set_to_none=True)
            s_e = rate(eager_fused, 50)
            legs["mapper_eager_fused"] = {"iterations_per_s": round(1.0 / s_e, 1), "ms_per_iteration": round(1e3 * s_e, 4)}
        # -- the mapper loop ACROSS keyframes [REF mp_Mapper.py:161-195, 244-245]: parameters + Adam state in a GaussianStore(stable=True),
        #    ONE captured graph with the live count on the device; every 10th iteration a keyframe appends 8 280 Gaussians (rows written in
        #    place, count bumped on the device), one prune in the middle.  The rate INCLUDES the ingestion and the prune; re-captures must be 0.
        if mg is not None and args.all_legs:
            from gs_icp_slam_amd.gaussian_store import GaussianStore
            from gs_icp_slam_amd.graph import MapperIterationGraph as _MG
            n_kf, per_kf = 12, 8280
            st = GaussianStore(P + (n_kf + 1) * per_kf, n_rest=0, stable=True)
            names = {"xyz": "means3D", "f_dc": "shs", "opacity": "opacities", "scaling": "scales", "rotation": "rotations"}

            def rows_of(src, lo, hi):
                d = {k: src[v][lo:hi].detach().to(dev).contiguous() for k, v in names.items()}
                d["f_rest"] = torch.zeros((hi - lo, 0, 3), device=dev)
                return d
            st.append(rows_of(raw, 0, P))
            kf_rows = [rows_of(raw, (i * per_kf) % (P - per_kf), (i * per_kf) % (P - per_kf) + per_kf) for i in range(n_kf)]
            for r_ in kf_rows:   # new surfels next to existing ones (shifted by 1 cm), as a keyframe's not-yet-mapped points would be
                r_["xyz"] = r_["xyz"] + 0.01
            opt_s = st.attach(FusedAdam, {"xyz": LRS["means3D"], "f_dc": LRS["shs"], "f_rest": LRS["shs"] / 20, "opacity": LRS["opacities"],
                                          "scaling": LRS["scales"], "rotation": LRS["rotations"]}, lr=0.0, eps=1e-15, capturable=True)
            ps = {v: st.params[k] for k, v in names.items()}
            mgs = _MG(ps, opt_s, H, W, cam["tanfovx"], cam["tanfovy"], sh_degree=0, capacity=int(capacity * 1.6), lambda_dssim=0.2, warmup=1,
                      live_count=st.live_count)
            mgs.set_view(rs.viewmatrix, rs.projmatrix, rs.campos, gt_color, gt_depth)
            mgs.capture()
            gobj = mgs.graph
            for _ in range(5):
                mgs.step()
            with torch.no_grad():   # one no-op prune first: the first call pays ~0.1 s of one-time torch kernel loading (the reference's own loop
                st.prune(torch.zeros(st.n, dtype=torch.bool, device=dev))   # prunes at iteration 0 as well [REF mp_Mapper.py:244])
            barrier()
            t0k = time.perf_counter()
            n_it = 0
            for kf_i in range(n_kf):
                st.append(kf_rows[kf_i])
                for _ in range(10):
                    mgs.set_view(rs.viewmatrix, rs.projmatrix, rs.campos, gt_color, gt_depth)
                    mgs.step()
                    n_it += 1
                if kf_i == n_kf // 2:
                    with torch.no_grad():
                        st.prune((torch.sigmoid(st.live("opacity")) < 0.005).squeeze(-1))
            barrier()
            dtk = time.perf_counter() - t0k
            # where the difference to mapper_only goes: the grown map's own iteration, one append, one prune (each measured alone, synchronised)
            t_it = rate(lambda: mgs.step(), 50)
            barrier(); ta = time.perf_counter(); st.append(kf_rows[0]); barrier(); t_app = time.perf_counter() - ta
            with torch.no_grad():
                rm = torch.zeros(st.n, dtype=torch.bool, device=dev)
                rm[-per_kf:] = True
            barrier(); tp = time.perf_counter(); st.prune(rm); barrier(); t_pr = time.perf_counter() - tp
            legs["mapper_with_keyframes"] = {"iterations_per_s": round(n_it / dtk, 1), "ms_per_iteration": round(1e3 * dtk / n_it, 4),
                                             "ms_per_iteration_at_final_size": round(1e3 * t_it, 4), "append_ms": round(1e3 * t_app, 3),
                                             "prune_ms": round(1e3 * t_pr, 3),
                                             "keyframes": n_kf, "gaussians_start": P, "gaussians_end": st.n, "prunes": 1,
                                             "graph_recaptures": 0 if mgs.graph is gobj else 1, "overflowed": bool(mgs.overflowed()),
                                             "what": "10 graph replays per keyframe; each keyframe appends 8 280 Gaussians in place (device-side live count), one prune"}
            del mgs, st, opt_s, ps
        # -- what UNMODIFIED mp_Mapper.py:219-248 executes on the drop-in rasteriser: torch activations [REF scene/gaussian_model.py:105-125],
        #    GaussianRasterizer's reference-compatible synchronous forward, torch l1 / ssim, loss.backward(), torch.optim.Adam, zero_grad
        rp = {k: v.to(dev).contiguous().requires_grad_(True) for k, v in raw.items()}
        topt = torch.optim.Adam([{"params": [rp[k]], "lr": lr, "name": k} for k, lr in LRS.items()], lr=0.0, eps=1e-15)
        window = _torch_window(3, dev)
        plain = GaussianRasterizer(rs)

        def reference_loop():
            means2D = torch.zeros_like(rp["means3D"], requires_grad=True) + 0
            depth, image, radii, used = plain(means3D=rp["means3D"], means2D=means2D, shs=rp["shs"], opacities=torch.sigmoid(rp["opacities"]),
                                              scales=torch.exp(rp["scales"]), rotations=torch.nn.functional.normalize(rp["rotations"]))
            mask = (gt_depth > 0.).detach()
            gt_im = gt_color * mask
            Ll1 = _torch_l1(image, gt_im)
            Ls = _torch_ssim(image, gt_im, window)
            Ld = _torch_l1(depth / 10.0, gt_depth / 10.0)
            loss = (1.0 - 0.2) * Ll1 + 0.2 * (1.0 - Ls) + 0.1 * Ld
            loss.backward()
            with torch.no_grad():
                topt.step()
                topt.zero_grad(set_to_none=True)
        s_r = rate(reference_loop, 30)
        legs["dropin_reference_loop"] = {"iterations_per_s": round(1.0 / s_r, 1), "ms_per_iteration": round(1e3 * s_r, 4),
                                         "what": "torch activations + synchronous GaussianRasterizer + torch l1/ssim + loss.backward() + torch.optim.Adam "
                                                 "(the statements of unmodified mp_Mapper.py:219-248)"}
        del rp, topt
        lap("mapper_legs")
        # -- the mapper iteration where D is REAL: the map the fused loop trains (5x the duplicates of the S-map surfels)
        if args.res == "replica" and os.environ.get("GSICP_BENCH_TRAINED_LEG", "1") != "0":
            try:
                legs["mapper_trained_map"] = trained_map_leg(dev, steps=100, reps=3, n_views=args.views)
            except Exception as e:   # noqa: BLE001 — a leg must not take the contract line with it
                legs["mapper_trained_map"] = {"status": "failed", "why": f"{type(e).__name__}: {e}"[:400]}
            lap("mapper_trained_map")
        # -- BASELINE configs[3]'s proxy: the same steady-state step at TUM's shape (640x480, 12 416-point noisy frames, gate 0.03, opacity threshold
        #    0.09 [REF tum.sh:135-142]) — a child run of this script, its contract line kept as the leg
        if args.res == "replica" and os.environ.get("GSICP_BENCH_CHILD") != "1" and os.environ.get("GSICP_BENCH_TUM_LEG", "1") != "0":
            import subprocess
            try:
                pr = subprocess.run([sys.executable, os.path.abspath(__file__), "--res", "tum", "--no-legs", "--no-cpu-baseline", "--full-line", "--legs-file", "/tmp/gsicp_bench_legs_tum_child.json", "--steps", str(args.steps),
                                     "--warmup", str(args.warmup), "--repeats", "3"], capture_output=True, text=True, timeout=300,
                                    env=dict(os.environ, GSICP_BENCH_CHILD="1"))
                line = [ln for ln in pr.stdout.splitlines() if ln.startswith("{")]
                tj = json.loads(line[-1])
                legs["step_tum"] = {k: tj.get(k) for k in ("value", "unit", "ms_per_step", "block_ms_per_step_p10_p50_p90", "pose_error_deg_mm", "stage_us_per_step")}
                legs["step_tum"].update(workload=tj["config"]["workload"], duplicates_per_view=tj["config"]["duplicates_per_view"],
                                        tracker_target_gaussians=tj["config"]["tracker_target_gaussians"])
            except Exception as e:   # noqa: BLE001
                legs["step_tum"] = {"status": "failed", "why": f"{type(e).__name__}: {e}"[:400]}
            lap("step_tum")

    # ---------------- CPU baseline: OpenMP GICP oracle (port), rank 0 only ----------------
    cpu = None
    if rank == 0 and world == 1 and not args.no_cpu_baseline and args.only != "mapper":     # (N = 1 only: at N > 1 the other ranks would wait 20 s at the next collective)
        import oracle
        oc = SteadyTracker(oracle.OracleGICP(), host=True) if steady else TrackerCase(args.pair, oracle.OracleGICP())
        oc.step()  # warm-up (thread pool, first touch)
        # the per-frame problem is small (8 k points): more OpenMP threads than it can feed only add overhead, so pick the
        # fastest thread count on this host first and report THAT as the baseline
        ncpu = os.cpu_count() or 1
        best_thr, best_rate = ncpu, 0.0
        for thr in sorted({t for t in (4, 8, 16, 32, 64, ncpu) if t <= ncpu}):
            oc.reg.set_num_threads(thr)
            oc.step()
            n, t0c = 0, time.perf_counter()
            while time.perf_counter() - t0c < 0.4:
                oc.step()
                n += 1
            r_ = n / (time.perf_counter() - t0c)
            if r_ > best_rate:
                best_thr, best_rate = thr, r_
        oc.reg.set_num_threads(best_thr)
        oc.k = 1 if steady else 0
        n, t_cpu0 = 0, time.perf_counter()
        while time.perf_counter() - t_cpu0 < args.cpu_seconds:
            To, _, _ = oc.step()
            n += 1
        t_cpu = time.perf_counter() - t_cpu0
        if steady:   # the same frame on both sides: poses must agree
            chk = SteadyTracker(pygicp.FastGICP())
            oc.k = chk.k = 3
            agree = bool(np.allclose(oc.step()[0], chk.step()[0], atol=1e-5))
            what = (f"{n} steady-state frames (set_input_source + set_source_filter + align + get_source_correspondence; every 10th exports the source covariances, every 40th "
                    f"rebuilds the target from host arrays: set_input_target + set_target_covariances_fromqs, kd-tree rebuild) against {oc.n_target} map Gaussians, "
                    f"{len(oc.frames[0]['points'])} points per frame, {oc.reg.iterations} LM iterations")
        else:
            agree = bool(np.allclose(To, last["T"], atol=1e-5)) if "T" in last else None
            what = (f"{n} x (set_input_source + align + get_source_correspondence) on the {args.pair} S-pair {args.res}, {len(trk.sp['points_b'])} points, "
                    f"{oc.reg.iterations} LM iterations")
        cpu = {"value": round(n / t_cpu, 2), "unit": "tracker frames/s (GICP only; the reference has no CPU rasteriser)",
               "cores": best_thr, "host_cores": ncpu, "kind": "port",
               "sample": what + f", {t_cpu:.1f} s wall, OpenMP kd-tree oracle at its fastest thread count",
               "pose_agrees_with_gpu": agree}

    lap("cpu_baseline")
    # ---------------- the reference's OWN two-process system on the drop-ins: BASELINE's metric as SURVEY 8(d) defines it ----------------
    # System FPS [REF mp_Tracker.py:333] and ATE (the reference's mean statistic [REF mp_Tracker.py:334, 479] and a true RMSE) of the unmodified
    # gs_icp_slam_unlimit.py on a 400-frame synthetic Replica-layout sequence, PSNR / SSIM of its end-of-run pass [REF mp_Mapper.py:335-422]
    ref_run = ref_run_fused = None
    noisy_runs = {}
    if rank == 0 and world == 1 and args.only is None and not args.no_reference_leg and not args.no_legs and os.environ.get("GSICP_BENCH_CHILD") != "1":
        import subprocess
        torch.cuda.synchronize()
        have_ref = os.path.exists(os.path.join(ROOT, "oracle", "_ref", "refpy", "mp_Mapper.pyc"))
        have_fused = os.path.exists(os.path.join(ROOT, "oracle", "_ref", "refpy_fused", "mp_Mapper.pyc"))

        def system_run(frames, extra=(), detail=True):
            """tools/run_reference_slam.py: the reference's unmodified gs_icp_slam_unlimit.py (byte-compiled by oracle/make_refpy.py in the build container) as the
            DRIVER of the three drop-in packages on a synthetic Replica-layout sequence; its own printed statistics come back as one JSON line."""
            t0r = time.perf_counter()
            if not have_ref:
                return {"status": "skipped", "why": "oracle/_ref/refpy is not on this box (python __graft_entry__.py builds it where /root/reference exists)"}
            try:
                pr = subprocess.run([sys.executable, os.path.join(ROOT, "tools", "run_reference_slam.py"), "--synthetic", str(frames), "--cache", "/tmp/gsicp_synth_cache",
                                     "--timeout", "240"] + list(extra), capture_output=True, text=True, timeout=420,
                                    env=dict(os.environ, **({"GSICP_ATE_DETAIL": "1"} if detail else {})))
                line = [ln for ln in pr.stdout.splitlines() if ln.startswith("{")]
                rj = json.loads(line[-1]) if line else {"status": "failed", "why": (pr.stderr or pr.stdout)[-400:]}
            except Exception as e:   # noqa: BLE001 — the reference run must not take the benchmark line with it
                rj = {"status": "failed", "why": f"{type(e).__name__}: {e}"}
            rj["leg_wall_s"] = round(time.perf_counter() - t0r, 1)
            return rj
        if not args.system_legs:
            ref_run = system_run(400)       # default: ONE clean run of the untouched system (System FPS / ATE / PSNR of the compact line; the same 400-frame
            #                                 sequence rounds 3-5 reported: a 200-frame run is dominated by the start-up of the three processes, 111 against 178 FPS)
        else:
            ref_run = system_run(400)
            # the same run with SURVEY 8(f)'s rows applied to the reference's files (oracle/make_refpy.py --fused; gs_icp_slam_amd/refglue.py)
            if have_fused:
                ref_run_fused = system_run(400, ["--fused"], detail=False)
            # the same pair on NOISY depth (sensor model sigma(z) = 1.2 mm + 1.9 mm (z - 0.4)^2, 15 % holes) with fast hand-held motion: the bar of VERDICT r4
            # item 1 — the fused system (default pacing: refglue.DEFAULT_ITERS_PER_FRAME) must keep the untouched system's ATE
            for fused_ in (False, True):
                if os.environ.get("GSICP_BENCH_NOISY_LEG", "1") == "0" or (fused_ and not have_fused):
                    continue
                noisy_runs["fused" if fused_ else "untouched"] = system_run(300, ["--noise", "--speed", "2", "--jitter", "0.003"] + (["--fused", "--policy", "freeze"] if fused_ else []))
        lap("reference_system_runs")

    # ---------------- multi-GPU bookkeeping ----------------
    ranks_seen = None
    if world > 1:
        props = torch.cuda.get_device_properties(dev)
        mine = f"rank {rank}: cuda:{dev_index} {props.name} uuid={getattr(props, 'uuid', '?')}"
        gathered = [None] * world
        dist.all_gather_object(gathered, mine)
        ranks_seen = gathered

    if rank == 0:
        ms = 1e3 * dt / args.steps
        headline_value, headline_scaling, headline_blocks = args.steps / dt, "strong", blocks
        if kf_leg is not None:
            legs = dict(legs or {})
            if args.mp_mode == "keyframes":       # the throughput mode is the headline; the tile-sharded (parity) mode becomes the leg
                legs["tile_sharded"] = {"mode": "tiles", "value": round(args.steps / dt, 3), "ms_per_step": round(ms, 4), "scaling": "strong",
                                        "block_ms_per_step": [round(1e3 * b / args.steps, 4) for b in blocks]}
                headline_value, headline_scaling, ms = kf_leg["value"], "weak", kf_leg["ms_per_step"]
                headline_blocks = [1e-3 * b * args.steps for b in kf_leg["block_ms_per_step"]]
            else:
                legs["keyframe_parallel"] = kf_leg
        stage_us = {k: round(v, 2) for k, v in per_launch_us.items()}
        it = align_stats.get("iterations")
        ang_mm = (tuple(trk.worst) if steady else trk.pose_error(last["T"])) if "T" in last else (None, None)
        bl = sorted(1e3 * b_ / args.steps for b_ in headline_blocks)
        pct = lambda q: round(bl[min(len(bl) - 1, int(round(q * (len(bl) - 1))))], 4)   # noqa: E731
        tkey = "steady" if steady else args.pair
        motions.setdefault("steady", "consecutive frames of the synthetic trajectory (~7 mm / 0.25 deg apart) against the map's trackable Gaussians; every 10th frame "
                                     "exports the source covariances, every 40th replaces the target (set_target_from_gaussians)")
        if "T" not in last:
            workload = f"{args.only} only"
        elif steady:
            workload = (f"BASELINE configs[2] shape, steady state: tracker frame = one of {len(trk.frames)} consecutive trajectory frames ({len(trk.sp['points_b'])} pts, gate "
                        f"{cfg['max_corr']} m, {it} LM iterations, worst pose error over the run {ang_mm[0]:.4f} deg / {ang_mm[1]:.2f} mm) against the {trk.n_target} trackable "
                        f"Gaussians of the S-map, mapping keyframe every {trk.map_kf} frames, tracking keyframe (target replaced on the device) every {trk.track_kf}; "
                        f"concurrent with one S-map mapper iteration (P={P}, {W}x{H}, sh_degree 0, depth = sum z alpha T, fromqs scale^2) on the next of {n_views} "
                        f"keyframe views (D = {min(D_views)}..{max(D_views)} duplicates)")
        else:
            workload = (f"BASELINE configs[2] shape: tracker frame on the {args.pair} S-pair {args.res} [{motions[args.pair]}; {len(trk.sp['points_b'])} pts, "
                        f"gate {cfg['max_corr']} m, {it} LM iterations, lands {ang_mm[0]:.3f} deg / {ang_mm[1]:.1f} mm from the true motion] concurrent with one "
                        f"S-map mapper iteration (P={P}, {W}x{H}, sh_degree 0, depth = sum z alpha T, fromqs scale^2) on the next of {n_views} keyframe views")
        rr = ref_run or {}
        if "T" not in last:
            workload_short = workload
        elif steady:
            workload_short = (f"Replica room0-shaped synthetic (BASELINE configs[2]), steady state: GICP tracker frame ({len(trk.sp['points_b'])} pts, gate {cfg['max_corr']} m, {it} LM it.) "
                              f"vs {trk.n_target} trackable map Gaussians, keyframes every {trk.map_kf}/{trk.track_kf} frames, concurrent with one mapper iteration "
                              f"(P={P}, {W}x{H}, sh 0) over {n_views} views")
        else:
            workload_short = (f"Replica room0-shaped synthetic (BASELINE configs[2]): GICP tracker frame on the {args.pair} S-pair ({len(trk.sp['points_b'])} pts, gate "
                              f"{cfg['max_corr']} m, {it} LM it.) concurrent with one mapper iteration (P={P}, {W}x{H}, sh 0) over {n_views} views")
        fused_pol = None
        if ref_run_fused is not None or noisy_runs.get("fused") is not None:
            from gs_icp_slam_amd.refglue import POLICY_NOTES
            fused_pol = {"reference_system_run_fused": POLICY_NOTES["free"], "reference_system_run_noisy_fused (ate_cm_noisy_fused)": POLICY_NOTES["freeze"]}
        out = {
            "metric": ("SLAM hot-path FPS (GICP tracker frame + one full mapper iteration: render, loss, backward, Adam), Replica room0-shaped synthetic"
                       if args.only is None else f"DIAGNOSTIC: {args.only} half only"),
            "value": round(headline_value, 3), "unit": "frames/s", "n_gpus": world, "steps": args.steps, "warmup": args.warmup,
            "ms_per_step": round(ms, 4), "higher_is_better": True, "scaling": headline_scaling if world > 1 else "strong", "vs_baseline": None, "dtype": "f32",
            "data": "synthetic",
            "repeats": len(headline_blocks), "timed_seconds": round(sum(headline_blocks), 3),
            "block_ms_per_step": [round(1e3 * b_ / args.steps, 4) for b_ in headline_blocks[:40]],
            "block_ms_per_step_p10_p50_p90": [pct(0.1), pct(0.5), pct(0.9)], "statistic": "mean over the timed blocks (all timed steps / all timed seconds)",
            # BASELINE's metric as SURVEY 8(d) defines it — what the reference ITSELF prints when its unmodified two-process system runs on the drop-ins
            # (400-frame synthetic Replica-layout sequence, gs_icp_slam_unlimit.py, replica.sh's flags); the whole record is legs.reference_system_run
            "system_fps": rr.get("system_fps"), "ate_cm": rr.get("ate_rmse_cm"), "ate_true_rmse_cm": rr.get("ate_true_rmse_cm"), "psnr": rr.get("psnr"),
            "ssim": rr.get("ssim"), "processes_that_loaded_it": rr.get("processes_that_loaded_it"),
            # the same system on noisy depth + fast motion (300 frames), untouched and with SURVEY 8(f)'s rows applied at the default pacing: the reference's
            # printed statistic (mean aligned error) and the true RMSE
            "ate_cm_noisy": noisy_runs.get("untouched", {}).get("ate_rmse_cm"), "ate_cm_noisy_fused": noisy_runs.get("fused", {}).get("ate_rmse_cm"),
            "ate_true_rmse_cm_noisy": noisy_runs.get("untouched", {}).get("ate_true_rmse_cm"),
            "ate_true_rmse_cm_noisy_fused": noisy_runs.get("fused", {}).get("ate_true_rmse_cm"),
            "fused_policy": fused_pol,
            "config": {"workload": workload, "workload_short": workload_short,
                       "tracker_workload": tkey, "tracker_motion": motions[tkey], "lm_iterations": it,
                       "tracker_target_gaussians": (trk.n_target if steady else None),
                       "gaussians": P, "width": W, "height": H, "duplicates_per_rank": D_local, "visible_gaussians": P_vis,
                       "keyframe_views": n_views, "duplicates_per_view": D_views, "visible_per_view": Pvis_views,
                       "tracker_mapper_overlap": worker is not None,
                       "step_coupling": ("free-running: K tracker frames and K mapper iterations run concurrently, each at its own pace; the block ends when both are done"
                                         if free_running else ("lockstep: both halves joined after every step" if worker is not None else "one half after the other")),
                       "mapper_iterations_in_flight": args.mapper_inflight, "cu_split": cu_split,
                       "mapper_iteration": (("one hipGraph replay per iteration" + (" (tile all-gather + gradient all-reduce captured inside)" if (world > 1 or force_coll) else ""))
                                            if mg is not None else ("eager launches from Python" if capture_error is None else f"eager (capture failed: {capture_error})")),
                       "rccl_graph_probe": rccl_graph_probe,
                       "exchange_bytes_per_rank": ({"image_all_gather_chunk": mg.rasterizer.holder.last_image_bytes,
                                                    "gradient_all_reduce_block": mg.rasterizer.holder.last_volume_bytes}
                                                   if (mg is not None and (world > 1 or force_coll)) else None),
                       "variants": {"depth_mode": "sum z alpha T (un-normalised)", "fromqs_scale_mode": "s^2", "regularization": "PLANE"},
                       "mp_mode": (args.mp_mode if (world > 1 or force_coll) else None),
                       "mp_bands": ({"mode": args.mp_bands, "super_tile_row_boundaries": bands} if world > 1 else None),
                       "parallelism": ("single GPU" if world == 1 else
                                       (f"mapper tiles sharded x{world} ({'collective' if backend != 'nccl' else 'RCCL'} "
                                        + ("all-gather of own tiles" if bands is None else "halo exchange between contiguous bands of super-tile rows")
                                        + " + all-reduce of visible gradient rows), tracker replicated"
                                        if args.mp_mode == "tiles" else
                                        f"data-parallel over keyframes x{world} (every rank its own view, one dense RCCL gradient all-reduce per step), tracker replicated")),
                       "world_size": world, "backend": backend if world > 1 else None, "rccl_ranks_seen": ranks_seen},
            "render_bwd_ms_per_iter": round(sum(v for k, v in per_launch_us.items() if not k.startswith(("gicp", "loss_", "adam"))) / 1e3, 4),
            "loss_adam_ms_per_iter": round(sum(v for k, v in per_launch_us.items() if k.startswith(("loss_", "adam"))) / 1e3, 4),
            "tracker_align_kernel_us": stage_us.get("gicp_align"),
            # steady: worst error over every frame tracked in the run.  (`--tracker pair --pair survey`, rounds 1-3: SURVEY 8(d)'s pair sits outside GICP's
            # basin at Replica's 2 cm gate — HIP and oracle alike converge to a wrong pose; it is legs.tracker_only_survey / legs.survey_pair_step now.)
            "pose_error_deg_mm": [round(ang_mm[0], 4), round(ang_mm[1], 3)] if "T" in last else None,
            "tracker_pose_is_the_true_motion": (bool(ang_mm[0] < 0.05 and ang_mm[1] < 1.0) if "T" in last else None),
            # what the UNMODIFIED mp_Mapper.py:219-248 statements cost on the drop-in rasteriser (the headline needs the fused, captured iteration)
            "dropin_reference_loop_ms_per_iteration": (legs or {}).get("dropin_reference_loop", {}).get("ms_per_iteration"),
            "stage_us_per_step": stage_us,
            "stage_us_source": ("one hipEvent bracket per kernel in EAGER iterations run right after the timed region (kernels inside a replayed hipGraph carry no "
                                "events): they read ~5-15 % above the same kernels inside the graph; the rocprofv3 kernel traces under profiles/ time the replayed kernels"),
            "legs": legs, "roofline": roofline, "roofline_longest_kernel": roofline_align, "cpu_baseline": cpu,
        }
        if ref_run is not None:
            out["legs"] = dict(out["legs"] or {}, reference_system_run=ref_run, reference_system_run_fused=ref_run_fused,
                               reference_system_run_noisy=noisy_runs.get("untouched"), reference_system_run_noisy_fused=noisy_runs.get("fused"))
        lap("bookkeeping")
        out["section_wall_s"] = dict(sect, total=round(sum(sect.values()), 1))
        # ---- the FULL record goes to a file next to this script; stdout carries ONE compact line (a 22 KB line was cut by the driver and parsed as nothing)
        legs_path = args.legs_file
        try:
            with open(legs_path, "w") as fh:
                json.dump(out, fh, indent=1)
        except OSError:
            legs_path = os.path.join("/tmp", "gsicp_bench_legs.json")
            with open(legs_path, "w") as fh:
                json.dump(out, fh, indent=1)
        print(json.dumps(out if args.full_line else compact_line(out, legs_path)))
    if worker is not None:
        jobs.put(None)
    if world > 1 or force_coll:
        for g_ in (mg, mgk):
            if g_ is not None:
                g_.release()      # a hipGraph that replays RCCL kernels must not outlive the communicator
        torch.cuda.synchronize()
        dist.destroy_process_group()


if __name__ == "__main__":
    sys.exit(main() or 0)
