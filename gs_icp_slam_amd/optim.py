"""Multi-tensor Adam in one HIP launch: a drop-in for the `torch.optim.Adam(l, lr=0.0, eps=1e-15)`
that GaussianModel builds [REF scene/gaussian_model.py:222-231] and the mapper steps [REF mp_Mapper.py:247].

State layout is torch's (`state[p] = {"step", "exp_avg", "exp_avg_sq"}`), because GaussianModel edits the optimiser state
in place when it appends or prunes Gaussians [REF scene/gaussian_model.py:409-492].  amsgrad / weight decay / maximize are
not supported (the reference does not use them).

``capturable=True`` (same meaning as torch.optim.Adam's flag) keeps the step count and the learning rates in device
memory, so that ``step()`` can be captured in a HIP graph and replayed (gs_icp_slam_amd/graph.py).  ``state[p]["step"]``
is then an int32 device tensor shared by the parameters that were first stepped together; after changing a group's
``lr`` call ``sync_lr()`` (outside capture) to push the new values to the device.

Beside it, for parameters of any number and of f32, bf16 or f16 (no reference counterpart: the reference trains with torch.optim.Adam):

    norm = grad_norm(grads)                                               # 2-norm over all of them, a device scalar
    adamw_step(params, grads, exp_avgs, exp_avg_sqs, lr=..., step=t)      # torch.optim.AdamW's step, one launch per 64 tensors
    adamw_step_8bit(params, grads, moments, block_exps, lr=..., step=t)   # the same with both moments in 8 bits
    exp_avgs, exp_avg_sqs = decode_moments(moments, block_exps)           # what 8-bit moments stand for

and `FusedAdamW`, the optimiser over them.  `max_norm=` clips by the global norm inside the step: the factor never leaves the device and the gradients are not rewritten.
"""
import array
import ctypes
import math

import torch

from . import _lib

_MAX = 8


def _counts_beside(step, p):
    """Whether a state's step count is what the capturable kernels read and advance: an int32 tensor on the parameter's device."""
    return torch.is_tensor(step) and step.dtype == torch.int32 and step.device == p.device


def _counter_beside(step, p, made):
    """A step count as that, wherever and whatever it was (a number, a tensor of a state that was loaded to the host, torch's float counter).  made: what the call has made so far;
    counters that were one tensor stay one, of others those that agree become one."""
    key = (step.data_ptr() if torch.is_tensor(step) and step.dtype == torch.int32 else int(step), p.device)
    if key not in made:
        made[key] = torch.full((), int(step), dtype=torch.int32, device=p.device)
    return made[key]


class FusedAdam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, capturable=False):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps))
        self.capturable = bool(capturable)
        self._lr_dev = {}       # (group index, position, betas, eps) bucket key -> [device double tensor, host lr values it holds]
        self._guard = None      # (count tensor uint32/int32[1], limit): skip the step when count > limit (capturable path)
        self.skipped_steps = None   # device int32[1], sticky: steps skipped by the guard since construction (read it whenever convenient)
        self._live_rows = None      # device int32[1]: parameters are capacity-backed, only this many leading rows are updated
        self._row_freeze = None     # (device int32[rows] mask, names of the param groups it applies to): rows with a non-zero word are left alone
        self._grad_rows = None      # device int32[rows] (the rasteriser's radii): rows with a word <= 0 take g = 0 and their gradient is not read
        self._prebumped = False     # the NEXT capturable step() finds its step counter already advanced (mapper_loss_and_grads(step_bump=...))

    def set_grad_row_mask(self, radii):
        """Capturable path, SPARSE gradients (round 6): `radii` = the int32 (P,) output of the rasteriser forward whose backward produced the gradients of
        the next step().  Rows with radii <= 0 are culled Gaussians: their gradient is zero by definition, the backward (GaussianRasterizationSettings.
        sparse_grads) did not write it and this step does not read it — the update is torch.optim.Adam's on g = 0.  Applies to every tensor with P rows;
        `None` removes it (every gradient element is read again).  Read at every step, so call it with the forward's radii before each step()."""
        if radii is not None and (not radii.is_cuda or radii.dtype != torch.int32 or not radii.is_contiguous()):
            raise RuntimeError("FusedAdam.set_grad_row_mask: expected the contiguous int32 device tensor `radii` of the rasteriser forward")
        self._grad_rows = radii

    def shared_step_tensor(self):
        """The ONE device step counter every parameter of this optimiser shares (capturable path, after the first step), or None when the parameters
        do not all share one — what mapper_loss_and_grads(step_bump=...) advances ahead of a step(step_already_bumped=True)."""
        steps = {}
        for group in self.param_groups:
            for p in group["params"]:
                st = self.state.get(p, {})
                if not _counts_beside(st.get("step"), p):
                    return None
                steps[st["step"].data_ptr()] = st["step"]
        return next(iter(steps.values())) if len(steps) == 1 else None

    def set_row_freeze(self, mask, group_names):
        """Capturable path: the param groups named in `group_names` (their "name" key, as GaussianModel sets it [REF scene/gaussian_model.py:222-229])
        leave the rows whose `mask` word (DEVICE int32, one per row, read at every step) is non-zero untouched — parameter and both moments, as if
        those rows were no parameters.  `mask=None` removes it.  (gsicp_adam_step_masked; used by refglue's `freeze` policy.)"""
        if mask is None:
            self._row_freeze = None
            return
        if not mask.is_cuda or mask.dtype != torch.int32 or not mask.is_contiguous():
            raise RuntimeError("FusedAdam.set_row_freeze: expected a contiguous int32 device tensor (one word per row)")
        self._row_freeze = (mask, frozenset(group_names))

    def scoped_bindings(self, guard=None, live_rows=None):
        """Context manager: bind an overflow guard and / or a live-row count for the launches issued inside (a graph capture), then restore
        what was bound before — so that eager steps on the same optimiser afterwards are not silently gated by a graph's last replay."""
        opt = self

        class _Scope:
            def __enter__(self_):
                self_.prev = (opt._guard, opt._live_rows)
                if guard is not None:
                    opt.set_overflow_guard(*guard)
                if live_rows is not None:
                    opt.set_live_rows(live_rows)
                return opt

            def __exit__(self_, *exc):
                opt._guard, opt._live_rows = self_.prev
                return False
        return _Scope()

    def set_live_rows(self, n_dev):
        """Capturable path: the parameter tensors are the full-capacity buffers of a preallocated map (GaussianStore); update only the
        first n_dev[0] rows of each.  n_dev changes on the device (append / prune) without any pointer or launch changing."""
        if n_dev is not None and (not n_dev.is_cuda or n_dev.dtype != torch.int32 or n_dev.numel() != 1):
            raise RuntimeError("FusedAdam.set_live_rows: expected an int32[1] device tensor")
        self._live_rows = n_dev

    def set_overflow_guard(self, count, limit):
        """Capturable path: skip the whole step (parameters, moments and step count untouched) whenever `count` (a DEVICE int32[1],
        e.g. GaussianRasterizer.num_rendered) exceeds `limit` (the rasteriser's list capacity) at the time the step runs — the
        sync-free forward then rendered nothing and every gradient is zero.  `skipped_steps` counts such steps on the device."""
        if count is None:
            self._guard = None
            return
        if not count.is_cuda or count.numel() != 1 or count.element_size() != 4:
            raise RuntimeError("FusedAdam.set_overflow_guard: count must be a 4-byte integer device tensor with one element")
        self._guard = (count, int(limit))
        if self.skipped_steps is None or self.skipped_steps.device != count.device:
            self.skipped_steps = torch.zeros(1, dtype=torch.int32, device=count.device)

    def sync_lr(self):
        """Push the param groups' current learning rates to the device arrays of the capturable path."""
        for key, entry in self._lr_dev.items():
            new = [float(self.param_groups[gi]["lr"]) for gi, _pi in key[0]]
            if new != entry[1]:
                entry[0].copy_(torch.tensor(new, dtype=torch.float64))
                entry[1] = new

    def _step_capturable(self, lib, prebumped=False):
        # bucket = tensors that share (betas, eps, step counter); identified by (param-group index, position) pairs, which stay valid when
        # a map store re-binds fresh Parameter objects into the same groups [REF scene/gaussian_model.py:409-492] (ids of dead objects
        # can be reused by CPython, group positions cannot)
        buckets = {}
        fresh, moved = {}, {}
        for gi, group in enumerate(self.param_groups):
            b1, b2 = group["betas"]
            for pi, p in enumerate(group["params"]):
                if p.grad is None:
                    continue
                if not p.is_cuda or p.dtype != torch.float32 or not p.is_contiguous() or not p.grad.is_contiguous():
                    raise RuntimeError("FusedAdam(capturable): parameters and gradients must be contiguous float32 on the HIP device")
                st = self.state[p]
                if not _counts_beside(st.get("step"), p) and torch.cuda.is_current_stream_capturing():      # state made now would live in the graph, unwritten
                    raise RuntimeError("FusedAdam(capturable): run one step() outside graph capture first (allocates the state)")
                if len(st) == 0:
                    if p.device not in fresh:
                        fresh[p.device] = torch.zeros((), dtype=torch.int32, device=p.device)
                    st["step"] = fresh[p.device]
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                elif not torch.is_tensor(st["step"]):
                    st["step"] = torch.full((), int(st["step"]), dtype=torch.int32, device=p.device)
                elif not _counts_beside(st["step"], p):
                    st["step"] = _counter_beside(st["step"], p, moved)
                buckets.setdefault((float(b1), float(b2), float(group["eps"]), st["step"].data_ptr()), []).append(
                    (p, p.grad, st["exp_avg"], st["exp_avg_sq"], float(group["lr"]), st["step"], (gi, pi)))
        capturing = torch.cuda.is_current_stream_capturing()
        # every distinct step tensor is bumped exactly once per step(): by the LAST launch that reads it
        last_of = {}
        launches = []
        for (b1, b2, eps, sp), items in buckets.items():
            for i in range(0, len(items), _MAX):
                launches.append((b1, b2, eps, sp, items[i:i + _MAX]))
                last_of[sp] = len(launches) - 1
        live_keys = set()
        for li, (b1, b2, eps, sp, items) in enumerate(launches):
            dev = items[0][0].device
            key = (tuple(t[6] for t in items), b1, b2, eps)
            live_keys.add(key)
            lrs = [t[4] for t in items]
            if key not in self._lr_dev:
                if capturing:
                    raise RuntimeError("FusedAdam(capturable): run one step() outside graph capture first (allocates the device lr array)")
                self._lr_dev[key] = [torch.tensor(lrs, dtype=torch.float64).to(dev), lrs]
            elif not capturing and self._lr_dev[key][1] != lrs:
                self._lr_dev[key][0].copy_(torch.tensor(lrs, dtype=torch.float64))
                self._lr_dev[key][1] = lrs
            lr_dev = self._lr_dev[key][0]
            guard_ptr, guard_lim, skip_ptr = None, 0, None
            if self._guard is not None and self._guard[0].device == dev:
                guard_ptr, guard_lim = ctypes.c_void_p(self._guard[0].data_ptr()), self._guard[1]
                skip_ptr = ctypes.c_void_p(self.skipped_steps.data_ptr())
            with torch.cuda.device(dev):
                stream = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
                n = len(items)
                P = (ctypes.c_void_p * n)(*[t[0].data_ptr() for t in items])
                G = (ctypes.c_void_p * n)(*[t[1].data_ptr() for t in items])
                M = (ctypes.c_void_p * n)(*[t[2].data_ptr() for t in items])
                V = (ctypes.c_void_p * n)(*[t[3].data_ptr() for t in items])
                N = (ctypes.c_longlong * n)(*[t[0].numel() for t in items])
                live_ptr, RW, freeze_ptr, FR = None, None, None, None
                freeze = self._row_freeze if (self._row_freeze is not None and self._row_freeze[0].device == dev) else None
                rows = self._grad_rows if (self._grad_rows is not None and self._grad_rows.device == dev) else None
                if rows is not None and any(t[0].dim() == 0 or t[0].shape[0] != rows.numel() for t in items):
                    raise RuntimeError("FusedAdam.set_grad_row_mask: every parameter must have one row per entry of the mask")
                if (self._live_rows is not None and self._live_rows.device == dev) or freeze is not None or rows is not None:
                    RW = (ctypes.c_int * n)(*[(t[0].numel() // t[0].shape[0]) if t[0].dim() > 0 and t[0].shape[0] > 0 else 0 for t in items])
                if self._live_rows is not None and self._live_rows.device == dev:
                    live_ptr = ctypes.c_void_p(self._live_rows.data_ptr())
                if freeze is not None:
                    flags = [1 if self.param_groups[t[6][0]].get("name") in freeze[1] else 0 for t in items]
                    for t, fl in zip(items, flags):
                        if fl and t[0].dim() > 0 and t[0].shape[0] > freeze[0].numel():
                            raise RuntimeError("FusedAdam.set_row_freeze: the mask has fewer words than the tensor has rows")
                    if any(flags):
                        freeze_ptr, FR = ctypes.c_void_p(freeze[0].data_ptr()), (ctypes.c_int * n)(*flags)
                bump = 2 if prebumped else int(last_of[sp] == li)       # 2: the counter was advanced ahead of this launch, in stream order
                _lib.check(lib.gsicp_adam_step_sparse(n, P, G, M, V, N, ctypes.c_void_p(lr_dev.data_ptr()), b1, b2, eps,
                                                      ctypes.c_void_p(items[0][5].data_ptr()), bump, guard_ptr, guard_lim,
                                                      skip_ptr, live_ptr, RW, freeze_ptr, FR, ctypes.c_void_p(rows.data_ptr()) if rows is not None else None,
                                                      stream), "gsicp_adam_step_sparse")
            _native_lists().wrote((None, [t[0] for t in items]), 1)      # autograd must notice when a backward meets one that it saved before
        # Device lr arrays are NEVER freed: a captured MapperIterationGraph holds their addresses, and an eager step() that happens
        # to see fewer gradients (zero_grad(set_to_none=True), different chunking) must not hand that memory back to the caching allocator
        # while a graph may still replay.  One entry is <= 8 doubles; the number of distinct buckets an optimiser ever sees is a handful.
        del live_keys

    @torch.no_grad()
    def step(self, closure=None, step_already_bumped=False):
        """step_already_bumped (capturable path): the device step counter was advanced ahead of this call, in stream order, by
        mapper_loss_and_grads(step_bump=(self.shared_step_tensor(), ...)) — the update uses the counter as it is and no bump launch follows."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        lib = _lib.load()
        if step_already_bumped and not self.capturable:
            raise RuntimeError("FusedAdam.step(step_already_bumped=True) needs capturable=True (a device step counter)")
        if self.capturable:
            self._step_capturable(lib, prebumped=bool(step_already_bumped))
            return loss
        buckets = {}   # (beta1, beta2, eps, step, device) -> list of (p, g, m, v, lr)
        for group in self.param_groups:
            b1, b2 = group["betas"]
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not p.is_cuda:
                    raise RuntimeError("FusedAdam (gfx950): parameters must live on the HIP device; there is no CPU path")
                if p.dtype != torch.float32 or not p.is_contiguous():
                    raise RuntimeError("FusedAdam: parameters must be contiguous float32")
                st = self.state[p]
                if len(st) == 0:
                    st["step"] = 0
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st["step"] = int(st["step"]) + 1
                g = p.grad if p.grad.is_contiguous() else p.grad.contiguous()
                buckets.setdefault((float(b1), float(b2), float(group["eps"]), st["step"], p.device), []).append(
                    (p, g.to(torch.float32), st["exp_avg"], st["exp_avg_sq"], float(group["lr"])))
        for (b1, b2, eps, step, dev), items in buckets.items():
            with torch.cuda.device(dev):
                stream = ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
                for i in range(0, len(items), _MAX):
                    chunk = items[i:i + _MAX]
                    n = len(chunk)
                    P = (ctypes.c_void_p * n)(*[t[0].data_ptr() for t in chunk])
                    G = (ctypes.c_void_p * n)(*[t[1].data_ptr() for t in chunk])
                    M = (ctypes.c_void_p * n)(*[t[2].data_ptr() for t in chunk])
                    V = (ctypes.c_void_p * n)(*[t[3].data_ptr() for t in chunk])
                    N = (ctypes.c_longlong * n)(*[t[0].numel() for t in chunk])
                    LR = (ctypes.c_float * n)(*[t[4] for t in chunk])
                    _lib.check(lib.gsicp_adam_step(n, P, G, M, V, N, LR, b1, b2, eps, step, stream), "gsicp_adam_step")
            _native_lists().wrote((None, [t[0] for t in items]), 1)
        return loss


# ------------------------------------------------------------------------------------------------ AdamW over many tensors
_BLOCK = 128                       # elements per base exponent of 8-bit moments
_tensor_lists = None


def _native_lists():
    global _tensor_lists
    if _tensor_lists is None:
        try:
            from . import _tensor_lists as module
        except ImportError as e:
            raise ImportError("gs_icp_slam_amd/_tensor_lists not found: build it with `python -m gs_icp_slam_amd.build`") from e
        _tensor_lists = module
    return _tensor_lists


def _pack(what, names, rules, *lists):
    """Lists of tensors, checked, as host arrays (csrc/tensor_lists.cpp) -> (device index, whether it is the current one, its current stream, n, address of the arrays, what
    keeps them and the tensors alive).  The arrays: n addresses per list, n element counts (8 bytes each), n dtype codes."""
    return _native_lists().pack(what, names, rules, *lists)


def _at(a):
    """Address of an array.array's items (the array must outlive the call), or None."""
    return None if a is None else a.buffer_info()[0]


def _doubles(what, name, value, n):
    if isinstance(value, (int, float)):
        return array.array("d", (value,)) * n
    try:
        a = array.array("d", value)
    except TypeError:                       # a scalar of another library
        return array.array("d", (float(value),)) * n
    if len(a) != n:
        raise RuntimeError(f"{what}: {name} is a number or one per tensor ({len(a)} for {n} tensors)")
    return a


def _call(name, device, current, *args):
    """The entry point `name` of the library with `device` current."""
    fn = getattr(_lib.load(), name)
    if current:
        rc = fn(*args)
    else:
        with torch.cuda.device(device):
            rc = fn(*args)
    if rc < 0:
        _lib.check(rc, name)


def _norm(what, device, current, stream, n, addresses, numels, codes, max_norm, rows=None):
    """-> (norm: 0-dim f32 on the device, buffer whose first word is the clip factor or None).  rows: address of a gsicp_adamw_device that says which rows do not count."""
    dev = torch.device("cuda", device)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    size = _lib.load().gsicp_grad_norm_scratch_bytes(n, numels, codes)
    buffer = clip = scratch = None
    if size or max_norm is not None:
        if max_norm is not None and not max_norm > 0.0:
            raise RuntimeError(f"{what}: max_norm must be positive")
        buffer = torch.empty(size + 8, dtype=torch.uint8, device=dev)
        clip = buffer.data_ptr()
        scratch = clip + 8
    out = (max_norm or 0.0, norm.data_ptr(), clip, scratch, stream)
    if rows is None:
        _call("gsicp_grad_norm", device, current, n, addresses, numels, codes, *out)
    else:
        _call("gsicp_grad_norm_rows", device, current, n, addresses, numels, codes, rows, *out)
    return norm, buffer


def grad_norm(tensors):
    """2-norm over all elements of `tensors` (f32, bf16 or f16, mixed, any sizes, contiguous, one device) as a 0-dim f32 tensor on their device; nothing synchronises.
    Squares and sums are taken in double and in a fixed order: the same tensors give the same bits."""
    device, current, stream, n, at, keep = _pack("grad_norm", ("tensors",), "p", tensors)
    return _norm("grad_norm", device, current, stream, n, at, at + 8 * n, at + 16 * n, None)[0]


_NAMES_32, _NAMES_8 = ("parameters", "gradients", "exp_avgs", "exp_avg_sqs"), ("parameters", "gradients", "moments", "block_exps")
_NAMES_32_MASTERS, _NAMES_8_MASTERS = _NAMES_32 + ("masters",), _NAMES_8 + ("masters",)


def _adamw(what, bits, params, grads, masters, first, second, lr, weight_decay, betas, eps, step, max_norm=None, clip=None, seed=0, place=None, device_form=None):
    """Checks, lays out and launches a step of either form; -> the norm or None.  clip: device address of a factor taken before (max_norm is then not looked at);
    device_form(): the gsicp_adamw_device of a captured step and what it points to."""
    if masters is None:
        device, current, stream, n, at, keep = _pack(what, _NAMES_32 if bits == 32 else _NAMES_8, "pgff" if bits == 32 else "pghb", params, grads, first, second)
        mast, numels = None, at + 32 * n
    else:
        device, current, stream, n, at, keep = _pack(what, _NAMES_32_MASTERS if bits == 32 else _NAMES_8_MASTERS, "pgffm" if bits == 32 else "pghbm", params, grads, first, second,
                                                     masters)
        mast, numels = at + 32 * n, at + 40 * n
    codes = numels + 8 * n
    step = int(step)
    if step > 0x7FFFFFFF:                       # the call below would take its low 32 bits
        raise RuntimeError(f"{what}: a step count has 31 bits")
    weight_decay = _doubles(what, "weight_decay", weight_decay, n)
    if device_form is None:
        lr, dev, dev_keep = _doubles(what, "lr", lr, n), None, None
    else:
        lr, (dev, dev_keep) = None, device_form()
    norm = buffer = None
    if clip is None and max_norm is not None:
        norm, buffer = _norm(what, device, current, stream, n, at + 8 * n, numels, codes, max_norm)
        clip = buffer.data_ptr()
    args = (n, at, at + 8 * n, mast, at + 16 * n, at + 24 * n, numels, codes, _at(lr), _at(weight_decay), betas[0], betas[1], eps, step)
    if bits == 32:
        _call("gsicp_adamw_step", device, current, *args, clip, dev, stream)
    else:
        _call("gsicp_adamw_step_8bit", device, current, *args, int(seed) & 0xFFFFFFFF, _at(place), clip, dev, stream)
    _tensor_lists.wrote(keep, 0b10001)        # parameters and masters: a backward may have saved them (no graph reaches the moments; each list of 64 costs 0.8 us)
    return norm


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, lr, step, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, masters=None, max_norm=None):
    """One torch.optim.AdamW step (amsgrad and maximize off) over all `params`, in place; one launch per 64 tensors.

    params, grads: lists of contiguous f32 / bf16 / f16 tensors on one device, a gradient of its parameter's dtype; exp_avgs, exp_avg_sqs: f32; masters: list of f32 tensors (or
    None entries) that take the update of 16-bit parameters, which then receive it rounded.  lr, weight_decay: a number, or one per tensor.  step: the 1-based count of this
    step.  max_norm: clip by the global norm of `grads` (torch.nn.utils.clip_grad_norm_'s factor; the gradients themselves stay as they are) — the norm is returned as a 0-dim
    tensor, else None.  No tensor that the step writes may overlap another.  In a captured graph the replays repeat this step count (FusedAdamW(capturable=True) counts on the
    device)."""
    params = list(params)
    if not params:
        return None
    return _adamw("adamw_step", 32, params, grads, masters, exp_avgs, exp_avg_sqs, lr, weight_decay, betas, eps, step, max_norm)


def adamw_step_8bit(params, grads, moments, block_exps, *, lr, step, seed=0, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, masters=None, max_norm=None):
    """adamw_step with both moments in 8 bits: moments[k] int16 of the parameter's number of elements, block_exps[k] int16[ceil(numel / 128)]; all zero before the first step
    (new_moments_8bit).  Moments are rounded stochastically; the random bits are a function of (seed, step, place in the list, element), so the same call gives the same bits."""
    params = list(params)
    if not params:
        return None
    return _adamw("adamw_step_8bit", 8, params, grads, masters, moments, block_exps, lr, weight_decay, betas, eps, step, max_norm, seed=seed)


def new_moments_8bit(param):
    """(moments, block_exps) of a parameter before its first step."""
    return (torch.zeros(param.shape, dtype=torch.int16, device=param.device),
            torch.zeros((param.numel() + _BLOCK - 1) // _BLOCK, dtype=torch.int16, device=param.device))


def decode_moments(moments, block_exps, dtype=torch.float32):
    """-> (exp_avgs, exp_avg_sqs): the values of 8-bit moments, lists of tensors of the moments' shapes in f32 or bf16 (which holds every code's value exactly)."""
    moments, block_exps = list(moments), list(block_exps)
    if not moments:
        return [], []
    if dtype not in (torch.float32, torch.bfloat16):
        raise RuntimeError("decode_moments: dtype is float32 or bfloat16")
    device, current, stream, n, at, keep = _pack("decode_moments", ("moments", "block_exps"), "cb", moments, block_exps)
    exp_avgs = [torch.empty(t.shape, dtype=dtype, device=t.device) for t in moments]
    exp_avg_sqs = [torch.empty(t.shape, dtype=dtype, device=t.device) for t in moments]
    m, v = (array.array("Q", [t.data_ptr() for t in ts]) for ts in (exp_avgs, exp_avg_sqs))
    _call("gsicp_adamw_decode", device, current, n, at, at + 8 * n, _at(m), _at(v), at + 16 * n, int(dtype == torch.bfloat16), stream)
    return exp_avgs, exp_avg_sqs


def gather_moments_8bit(moments, block_exps, index, out=None):
    """Rows of 8-bit moments, as `t[index]` would take them from their values: -> (moments, block_exps), lists of new tensors (or `out`, two lists of contiguous int16 tensors that
    hold at least that much; nothing behind it is written).  All tensors have the same number of rows; index: int64 on their device, rows outside come out zero.  Values are moved
    exactly, except those that fall below the smallest code of the 128-element block they come into (first moments become zero, second that code)."""
    moments, block_exps = list(moments), list(block_exps)
    if not moments:
        return [], []
    what = "gather_moments_8bit"
    device, current, stream, n, at, keep = _pack(what, ("moments", "block_exps"), "cb", moments, block_exps)
    dev = moments[0].device
    rows = moments[0].shape[0] if moments[0].dim() else -1
    if any(t.dim() == 0 or t.shape[0] != rows for t in moments):
        raise RuntimeError(f"{what}: every tensor must have the same number of rows")
    if index.dtype != torch.int64 or index.device != dev or index.dim() != 1 or not index.is_contiguous():
        raise RuntimeError(f"{what}: index must be a contiguous one-dimensional int64 tensor on the device of the moments")
    count = index.numel()
    widths = array.array("q", [math.prod(t.shape[1:]) for t in moments])
    if out is None:
        out = ([torch.empty((count,) + tuple(t.shape[1:]), dtype=torch.int16, device=dev) for t in moments],
               [torch.empty((count * w + _BLOCK - 1) // _BLOCK, dtype=torch.int16, device=dev) for w in widths])
    else:
        for ts, need in ((out[0], [count * w for w in widths]), (out[1], [(count * w + _BLOCK - 1) // _BLOCK for w in widths])):
            if len(ts) != n or any(t.dtype != torch.int16 or t.device != dev or not t.is_contiguous() or t.numel() < k for t, k in zip(ts, need)):
                raise RuntimeError(f"{what}: out must be contiguous int16 tensors on the device of the moments, large enough")
    if rows == 0:
        for ts, need in zip(out, ([count * w for w in widths], [(count * w + _BLOCK - 1) // _BLOCK for w in widths])):
            for t, k in zip(ts, need):
                t.view(-1)[:k].zero_()
        return out
    o_c, o_x = (array.array("Q", [t.data_ptr() for t in ts]) for ts in out)
    _call("gsicp_adamw_gather_rows", device, current, n, at, at + 8 * n, _at(o_c), _at(o_x), _at(widths), index.data_ptr(), count, rows, stream)
    return out


class FusedAdamW(FusedAdam):
    """torch.optim.AdamW (amsgrad and maximize off) over any number of f32, bf16 and f16 parameters, one launch per 64 of them with the same betas, eps and step count.

    state_bits      32: state[p] = {"step", "exp_avg", "exp_avg_sq"} (f32; torch's layout, so GaussianStore and the reference's append / prune keep working)
                    8: state[p] = {"step", "moments", "block_exps"} — adamw_step_8bit's; `moments(p)` gives their values.  For a map that grows or is pruned:
                    GaussianStore(moment_bits=8)
    master_weights  16-bit parameters keep an f32 copy in state[p]["master"] that takes the update
    max_grad_norm   clip by the global norm of all gradients of the step; `last_grad_norm` is then a 0-dim device tensor.  Rows that the step leaves alone (set_live_rows,
                    set_row_freeze) do not count, whatever their gradients hold
    seed            of the stochastic rounding of 8-bit moments
    capturable      as in FusedAdam: step count and learning rates on the device, the step can be captured and replayed; weight decay, betas and max_grad_norm are part of the
                    capture.  MapperIterationGraph takes it wherever it takes FusedAdam."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, capturable=False, state_bits=32, master_weights=False, max_grad_norm=None, seed=0):
        if state_bits not in (8, 32):
            raise ValueError("FusedAdamW: state_bits is 32 or 8")
        if not (lr >= 0.0 and eps >= 0.0 and weight_decay >= 0.0 and 0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError("FusedAdamW: lr, eps and weight_decay are not negative, betas in [0, 1)")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError("FusedAdamW: max_grad_norm must be positive")
        super().__init__(params, lr=lr, betas=betas, eps=eps, capturable=capturable)
        self.defaults["weight_decay"] = weight_decay
        for group in self.param_groups:
            group.setdefault("weight_decay", weight_decay)
        self.state_bits, self.master_weights, self.max_grad_norm, self.seed = state_bits, bool(master_weights), max_grad_norm, int(seed)
        self.last_grad_norm = None

    def set_live_rows(self, n_dev):
        """As in FusedAdam; with 8-bit moments the codes of the rows behind the live ones must be zero (as GaussianStore keeps them): they share the last live block's exponents."""
        super().set_live_rows(n_dev)

    def set_row_freeze(self, mask, group_names):
        if mask is not None and self.state_bits == 8:
            raise RuntimeError("FusedAdamW(state_bits=8): frozen rows need 32-bit moments (they would share block exponents with rows that move)")
        super().set_row_freeze(mask, group_names)

    def moments(self, p):
        """(exp_avg, exp_avg_sq) of a parameter that has been stepped, in f32, whatever state_bits is (a copy with 8, the state itself with 32)."""
        st = self.state.get(p)
        if not st:
            raise RuntimeError("FusedAdamW.moments: this parameter has not been stepped")
        if self.state_bits == 32:
            return st["exp_avg"], st["exp_avg_sq"]
        (m,), (v,) = decode_moments([st["moments"]], [st["block_exps"]])
        return m, v

    def load_state_dict(self, state_dict):
        """torch's load casts every state tensor to its parameter's dtype; moments, masters and 8-bit codes keep their own here, and parameters that shared a step counter
        share it again (those of torch's optimisers, which count per parameter, share one where they agree).  Masters are kept as this optimiser has them: those that the state lacks are made from the parameters (load these first), others are dropped.  A state of FusedAdam, which has no weight decay, leaves that of each group as it is here.  States of torch.optim.Adam and
        AdamW are taken, but not with amsgrad, maximize or a weight decay that is added to the gradient."""
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        names = ("exp_avg", "exp_avg_sq") if self.state_bits == 32 else ("moments", "block_exps")
        for i in saved:
            if any(k not in state_dict["state"].get(i, dict.fromkeys(names)) for k in names):
                raise ValueError(f"FusedAdamW(state_bits={self.state_bits}): the state was saved with another width of the moments")
        for g in state_dict["param_groups"]:
            for k, wanted in (("amsgrad", False), ("maximize", False), ("decoupled_weight_decay", True)):
                if bool(g.get(k, wanted)) != wanted and (k != "decoupled_weight_decay" or g.get("weight_decay", 0) != 0):
                    raise ValueError(f"FusedAdamW: the state was saved with {k}={g[k]}")
        decays = [g["weight_decay"] for g in self.param_groups]
        super().load_state_dict(state_dict)
        for g, decay in zip(self.param_groups, decays):     # FusedAdam's groups have none
            g.setdefault("weight_decay", decay)
        steps = {}
        for i, p in zip(saved, [p for g in self.param_groups for p in g["params"]]):
            for k, v in state_dict["state"].get(i, {}).items():
                if k == "step":
                    if self.capturable:
                        v = _counter_beside(v, p, steps)
                    else:
                        v = int(v)
                elif torch.is_tensor(v):
                    v = v.detach().to(device=p.device, copy=True)
                self.state[p][k] = v
            st = self.state.get(p)
            if st:
                if not self.master_weights or p.dtype == torch.float32:
                    st.pop("master", None)
                elif "master" not in st:
                    st["master"] = p.detach().float()

    def _new_state(self, p, step):
        st = self.state[p]
        st["step"] = step
        if self.state_bits == 32:
            st["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            st["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        else:
            st["moments"], st["block_exps"] = new_moments_8bit(p)
        if self.master_weights and p.dtype != torch.float32:
            st["master"] = p.detach().float()

    @torch.no_grad()
    def step(self, closure=None, step_already_bumped=False):
        """step_already_bumped: as in FusedAdam.step."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if step_already_bumped and not self.capturable:
            raise RuntimeError("FusedAdamW.step(step_already_bumped=True) needs capturable=True (a device step counter)")
        buckets, fresh, moved, place, may_run = {}, {}, {}, -1, self.capturable
        for gi, group in enumerate(self.param_groups):
            b1, b2 = group["betas"]
            for pi, p in enumerate(group["params"]):
                place += 1                                  # counts every parameter: the random bits of one do not depend on which others have a gradient
                if p.grad is None:
                    continue
                if not p.is_cuda:
                    raise RuntimeError("FusedAdamW (gfx950): parameters must live on the HIP device; there is no CPU path")
                if not may_run:
                    if torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("FusedAdamW: capturing a step needs capturable=True (the replays would repeat one step count)")
                    may_run = True
                if p.grad.is_sparse:
                    raise RuntimeError("FusedAdamW: sparse gradients are not supported")
                st = self.state[p]
                if self.capturable and not _counts_beside(st.get("step"), p) and torch.cuda.is_current_stream_capturing():      # as in FusedAdam
                    raise RuntimeError("FusedAdamW(capturable): run one step() outside graph capture first (allocates the state)")
                if not st:
                    if self.capturable and p.device not in fresh:
                        fresh[p.device] = torch.zeros((), dtype=torch.int32, device=p.device)
                    self._new_state(p, fresh[p.device] if self.capturable else 0)
                elif self.capturable and not _counts_beside(st["step"], p):
                    st["step"] = _counter_beside(st["step"], p, moved)
                key = (float(b1), float(b2), float(group["eps"]), st["step"].data_ptr() if self.capturable else int(st["step"]), p.device)
                buckets.setdefault(key, []).append((p, p.grad.contiguous(), st, gi, pi, place))
        clip = buffer = None
        if self.max_grad_norm is not None and buckets:
            if self._grad_rows is not None:
                raise RuntimeError("FusedAdamW: max_grad_norm reads every gradient row, set_grad_row_mask says some were not written")
            if len({key[4] for key in buckets}) > 1:
                raise RuntimeError("FusedAdamW(max_grad_norm): the parameters live on several devices")
            items = [t for ts in buckets.values() for t in ts]
            device, current, stream, n, at, keep = _pack("FusedAdamW", ("gradients",), "p", [t[1] for t in items])
            rows, rows_keep = None, []
            if self.capturable:                             # rows that the step leaves alone do not count
                d = _lib.AdamWDevice()
                rows_keep = [d]
                if self._row_form(d, items, items[0][0].device, rows_keep):
                    rows = ctypes.addressof(d)
            self.last_grad_norm, buffer = _norm("FusedAdamW", device, current, stream, n, at, at + 8 * n, at + 16 * n, self.max_grad_norm, rows)
            clip = buffer.data_ptr()
        last_of = {key[3:]: key for key in buckets}         # a device counter is advanced by the last launch that reads it
        first, second = ("exp_avg", "exp_avg_sq") if self.state_bits == 32 else ("moments", "block_exps")
        for key, items in buckets.items():
            groups = [self.param_groups[t[3]] for t in items]
            masters = [t[2].get("master") for t in items]
            device_form = None
            if self.capturable:
                bump = 2 if step_already_bumped else int(last_of[key[3:]] == key)
                device_form = lambda items=items, key=key, bump=bump: self._device_form(items, key, bump)   # noqa: E731
            _adamw("FusedAdamW", self.state_bits, [t[0] for t in items], [t[1] for t in items], masters if any(m is not None for m in masters) else None,
                   [t[2][first] for t in items], [t[2][second] for t in items], [float(g["lr"]) for g in groups], [float(g["weight_decay"]) for g in groups], key[:2], key[2],
                   1 if self.capturable else key[3] + 1, clip=clip, seed=self.seed, place=array.array("i", [t[5] for t in items]), device_form=device_form)
            if not self.capturable:
                for t in items:
                    t[2]["step"] = key[3] + 1
        return loss

    def _device_form(self, items, key, bump):
        """The gsicp_adamw_device of one captured launch sequence, and the host arrays it points to."""
        device = key[4]
        ids = tuple((t[3], t[4]) for t in items)
        lrs = [float(self.param_groups[gi]["lr"]) for gi, _ in ids]
        entry = self._lr_dev.get((ids,) + key[:3])
        capturing = torch.cuda.is_current_stream_capturing()
        if entry is None:
            if capturing:
                raise RuntimeError("FusedAdamW(capturable): run one step() outside graph capture first (allocates the device lr array)")
            entry = self._lr_dev[(ids,) + key[:3]] = [torch.tensor(lrs, dtype=torch.float64).to(device), lrs]
        elif not capturing and entry[1] != lrs:
            entry[0].copy_(torch.tensor(lrs, dtype=torch.float64))
            entry[1] = lrs
        d = _lib.AdamWDevice(lr_dev=entry[0].data_ptr(), step_dev=key[3], bump_step=bump)
        keep = [d]
        if self._guard is not None and self._guard[0].device == device:
            d.guard_count, d.guard_limit, d.skipped = self._guard[0].data_ptr(), self._guard[1], self.skipped_steps.data_ptr()
        self._row_form(d, items, device, keep)
        return ctypes.addressof(d), keep

    def _row_form(self, d, items, device, keep):
        """Writes the live rows and row masks that apply to the tensors of `items` into d (its host arrays go to `keep`); -> whether there are any."""
        live = self._live_rows if self._live_rows is not None and self._live_rows.device == device else None
        freeze = self._row_freeze if self._row_freeze is not None and self._row_freeze[0].device == device else None
        rows = self._grad_rows if self._grad_rows is not None and self._grad_rows.device == device else None
        if live is None and freeze is None and rows is None:
            return False
        params = [t[0] for t in items]
        if rows is not None and any(p.dim() == 0 or p.shape[0] != rows.numel() for p in params):
            raise RuntimeError("FusedAdamW.set_grad_row_mask: every parameter must have one row per entry of the mask")
        width = array.array("i", [p.numel() // p.shape[0] if p.dim() > 0 and p.shape[0] > 0 else 0 for p in params])
        keep.append(width)
        d.row_width = _at(width)
        if live is not None:
            d.live_rows = live.data_ptr()
        if rows is not None:
            d.grad_rows = rows.data_ptr()
        if freeze is not None:
            flags = array.array("i", [int(self.param_groups[t[3]].get("name") in freeze[1]) for t in items])
            if any(fl and p.dim() > 0 and p.shape[0] > freeze[0].numel() for fl, p in zip(flags, params)):
                raise RuntimeError("FusedAdamW.set_row_freeze: the mask has fewer words than the tensor has rows")
            if any(flags):
                keep.append(flags)
                d.row_freeze, d.group_frozen = freeze[0].data_ptr(), _at(flags)
        return True
