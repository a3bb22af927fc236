"""Cases for measuring the optimiser operators of gs_icp_slam_amd.optim: the AdamW step over many tensors with its moments in 32 bits or in 8, and the
global gradient norm that clips it.

A case names an operator, a set of tensors and their type.  The tensors of a case are views of one flat buffer (each begins at a multiple of 128 elements, the
gaps hold zeros), so that the plain form is a handful of elementary torch operations over the whole buffer, whatever the number of tensors.

8-bit moments.  Two bytes per element and two per block of 128 consecutive elements of a tensor:
  moments     int16: low byte = sign (bit 7) and magnitude code (7 bits) of the first moment, high byte = code of the second moment
  block_exps  int16: low byte = base exponent bm of the block's first moments, high byte = base exponent bv of its second moments
A code c > 0 with base b stands for (1 + (c & 7) / 8) * 2^((c >> 3) + b - 127), 0 for zero; magnitude 127 is NaN, second-moment code 255 is infinity.
A block's base is the exponent of its largest finite value less 14 (first moments) or 30 (second), at least 1.  Values are rounded to a code
stochastically: random bits are a function of (seed, step, place of the tensor in the list, element), so they are inputs.
"""
import torch

own = False

BLOCK = 128
BETAS = (0.9, 0.999)
STEP0 = 100                      # steps taken before the measured one: bias corrections neither vanish nor dominate
G1, G2, G3, G4 = 0x9E3779B1, 0x85EBCA6B, 0x7FEB352D, 0x846CA68B
LANE = (0x6A09E667, 0xBB67AE85, 0x3C6EF373, 0xA54FF53B, 0x510E527F, 0x9B05688D, 0x1F83D9AB, 0x5BE0CD19)
M32 = 0xFFFFFFFF
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the AdamW step, moments in 32 bits
        # camera poses and exposure matrices of a window of 32 keyframes: 64 tensors of 7 and 12 numbers, pure latency
        dict(name="adamw_poses_32", op="adamw", layout="poses", count=32, dtype="float32", master=False, max_norm=0.0),
        # a young map: 40 k Gaussians, colours without higher harmonics
        dict(name="adamw_map_40k", op="adamw", layout="map", count=40000, rest=0, dtype="float32", master=False, max_norm=0.0),
        # the benchmark's map size with harmonics of degree 3, an odd row count, clipped
        dict(name="adamw_map_300k_sh3_clip", op="adamw", layout="map", count=300007, rest=15, dtype="float32", master=False, max_norm=0.1),
        # a network in bfloat16 with 32-bit masters, clipped
        dict(name="adamw_net_bf16_clip", op="adamw", layout="net", count=8, width=1024, dtype="bfloat16", master=True, max_norm=1.0),
        # a large map: 4 M Gaussians of degree 3
        dict(name="adamw_map_4m_sh3", op="adamw", layout="map", count=4000000, rest=15, dtype="float32", master=False, max_norm=0.0),
        # the AdamW step, moments in 8 bits
        dict(name="adamw8_poses_32", op="adamw8", layout="poses", count=32, dtype="float32", master=False, max_norm=0.0),
        dict(name="adamw8_map_300k_sh3", op="adamw8", layout="map", count=300007, rest=15, dtype="float32", master=False, max_norm=0.0),
        dict(name="adamw8_net_bf16_clip", op="adamw8", layout="net", count=8, width=512, dtype="bfloat16", master=True, max_norm=1.0),
        # the capacity of the reference's shared buffers: 10 M Gaussians
        dict(name="adamw8_map_10m", op="adamw8", layout="map", count=10000000, rest=0, dtype="float32", master=False, max_norm=0.0),
        # the global norm alone
        dict(name="norm_poses_32", op="norm", layout="poses", count=32, dtype="float32"),
        dict(name="norm_map_300k", op="norm", layout="map", count=300007, rest=0, dtype="float32"),
        dict(name="norm_net_fp16", op="norm", layout="net", count=8, width=1024, dtype="float16"),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    op = rng.choice(["adamw", "adamw", "adamw8", "adamw8", "norm"])
    layout = rng.choice(["poses", "map", "map", "net"])
    if layout == "poses":
        c = dict(op=op, layout=layout, count=spread(1, 200), dtype="float32")
    elif layout == "map":
        c = dict(op=op, layout=layout, count=spread(1000, 1500000), rest=rng.choice([0, 3, 8, 15]), dtype="float32")
    else:
        c = dict(op=op, layout=layout, count=rng.randint(1, 6), width=rng.randrange(65, 1000), dtype=rng.choice(["float32", "bfloat16", "float16"]))
    if op != "norm":
        c["master"] = c["dtype"] != "float32" and rng.random() < 0.7
        c["max_norm"] = rng.choice([0.0, 0.1, 1.0])
    return c


def tensors(case):
    """[(elements, learning rate, weight decay, gradient scale)] of a case, in the order of the parameter list."""
    n = case["count"]
    if case["layout"] == "poses":
        return [x for _ in range(n) for x in ((7, 1e-3, 0.0, 1e-2), (12, 2e-3, 1e-4, 1e-3))]
    if case["layout"] == "map":      # xyz, f_dc, f_rest (empty without higher harmonics), opacity, scaling, rotation, with the mapper's learning rates
        return [(3 * n, 1.6e-4, 0.0, 1e-4), (3 * n, 2.5e-3, 0.0, 1e-5), (3 * case["rest"] * n, 1.25e-4, 1e-2, 1e-6), (n, 5e-2, 1e-3, 1e-5), (3 * n, 5e-3, 0.0, 1e-5),
                (4 * n, 1e-3, 0.0, 1e-5)]
    d = case["width"]
    layer = [(d, 3e-4, 0.0, 1e-3)] + 4 * [(d * d, 3e-4, 0.1, 1e-4)] + [(d, 3e-4, 0.0, 1e-3), (4 * d * d, 3e-4, 0.1, 1e-4), (4 * d, 3e-4, 0.0, 1e-3), (4 * d * d, 3e-4, 0.1, 1e-4),
                                                                       (d, 3e-4, 0.0, 1e-3)]
    return [(32003 * d if case["width"] >= 512 else 4001 * d, 3e-4, 0.1, 1e-4)] + n * layer


def work(case):
    n = sum(t[0] for t in tensors(case))
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "norm":
        return {"bytes": n * size + 4, "flops": 2 * n}
    param = (size + 8) if case["master"] else 2 * size                   # with a master the parameter is only written
    if case["op"] == "adamw":
        return {"bytes": n * (param + size + 16), "flops": 16 * n}
    return {"bytes": n * (param + size + 4 + 4 / BLOCK + 4), "flops": 40 * n}      # codes in and out, and the moments' values handed out (2 x 16 bits)


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = "cuda"
    dt = TYPES[case["dtype"]]
    ts = tensors(case)
    gen = torch.Generator(device=dev).manual_seed(seed * 2 + 1)
    blocks = [-(-t[0] // BLOCK) for t in ts]
    first = [sum(blocks[:k]) for k in range(len(ts))]
    nb = sum(blocks)
    reps = torch.tensor(blocks, device=dev)

    def column(values, dtype=torch.float64):
        return torch.repeat_interleave(torch.tensor(values, dtype=dtype, device=dev), reps, output_size=nb).view(-1, 1)

    def normal():
        return torch.randn(nb, BLOCK, device=dev, generator=gen)

    at = torch.arange(nb, device=dev).view(-1, 1) - column(first, torch.int64)          # block within its tensor
    lane = torch.arange(BLOCK, device=dev).view(1, -1)
    real = at * BLOCK + lane < column([t[0] for t in ts], torch.int64)                  # not in a gap between two tensors
    scale = column([t[3] for t in ts]).float()
    # gradients spread over some orders of magnitude inside a block; of a map, most Gaussians are out of view in any one iteration: their gradient is zero
    spread = torch.exp(normal())
    seen = torch.rand(nb, BLOCK, device=dev, generator=gen)
    live = real & (seen < 0.35) if case["layout"] == "map" else real
    s = {"case": dict(case), "step": STEP0, "seed": 20 + seed}
    s["grads"] = torch.where(live, normal() * spread * scale, torch.zeros((), device=dev)).to(dt).view(-1)
    views = lambda flat: [flat[b * BLOCK: b * BLOCK + t[0]] for b, t in zip(first, ts)]      # noqa: E731
    s["grad_list"] = views(s["grads"])
    if case["op"] == "norm":
        return s
    weights = torch.where(real, normal(), torch.zeros((), device=dev)).view(-1)
    s["params"] = weights.to(dt)
    s["param_list"] = views(s["params"])
    s["masters"] = weights if case["master"] else None
    s["master_list"] = views(weights) if case["master"] else None
    born = real & (seen < 0.9) if case["layout"] == "map" else real                     # the newest Gaussians have no moments yet
    m = torch.where(born, 0.3 * normal() * spread * scale, torch.zeros((), device=dev))
    v = torch.where(born, (0.5 + seen) * spread.square() * scale.square(), torch.zeros((), device=dev))
    s["lr"], s["weight_decay"] = [t[1] for t in ts], [t[2] for t in ts]
    s["lr_column"], s["decay_column"] = column(s["lr"]), column(s["weight_decay"])
    s["eps"] = 1e-15 if case["layout"] == "map" else 1e-8
    if case["op"] == "adamw":
        s["exp_avg"], s["exp_avg_sq"] = m.view(-1), v.view(-1)
        s["exp_avg_list"], s["exp_avg_sq_list"] = views(s["exp_avg"]), views(s["exp_avg_sq"])
        return s
    s["place"] = column(list(range(len(ts))), torch.int64)
    s["lane"] = torch.tensor(LANE, dtype=torch.int64, device=dev)
    s["octet"] = at * (BLOCK // 8) + torch.arange(BLOCK // 8, device=dev).view(1, -1)
    s["moments"], s["block_exps"] = encode(m, v, *random_words(s, STEP0))
    s["moment_list"] = views(s["moments"])
    s["block_exp_list"] = [s["block_exps"][b: b + k] for b, k in zip(first, blocks)]
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def mix(x):
    x = (x ^ (x >> 16)) * G3 & M32
    x = (x ^ (x >> 15)) * G4 & M32
    return x ^ (x >> 16)


def random_words(s, step):
    """The 16 random bits of every first and every second moment of this step: one hashed word per octet, times an odd constant per element of it."""
    key = mix((s["seed"] + step * G1 + s["place"] * G2) & M32)
    word = mix(s["octet"] ^ key)
    r = (word.unsqueeze(2) * s["lane"] & M32).view(word.shape[0], BLOCK)
    return (r & 0xFFFF).int(), (r >> 16).int()


def base_exponent(bits, below):
    top = torch.where(bits < 0x7F800000, bits, 0).amax(1, keepdim=True)
    return ((top >> 23) - below).clamp_min(1)


def encode(m, v, um, uv):
    mb, vb = m.view(torch.int32) & 0x7FFFFFFF, v.view(torch.int32) & 0x7FFFFFFF
    bm, bv = base_exponent(mb, 14), base_exponent(vb, 30)
    low = ((bm << 23) + (1 << 20)).view(torch.float32)                   # the smallest magnitude that has a code
    mc = ((mb + (um << 4) + 8) >> 20) - (bm << 3)
    mc = torch.where(m.abs() < low, (m.abs() > low * 2.0 ** -16 * (um.float() + 0.5)).int(), mc)
    mc = torch.where(mc > 0, mc | ((m < 0).int() << 7), 0)
    mc = torch.where(mb >= 0x7F800000, 127, mc)
    vc = (((vb + (uv << 4) + 8) >> 20) - (bv << 3)).clamp_min(1)         # what is not zero stays so: the denominator must not vanish
    vc = torch.where(vb == 0, 0, torch.where(vb >= 0x7F800000, 255, vc))
    return (mc | (vc << 8)).short().view(-1), (bm | (bv << 8)).short().view(-1)


def decode(moments, block_exps):
    c, b = moments.view(-1, BLOCK).int(), block_exps.view(-1, 1).int()
    mc, vc, bm, bv = c & 0x7F, (c >> 8) & 0xFF, b & 0xFF, (b >> 8) & 0xFF
    m = ((mc << 20) + (bm << 23)).view(torch.float32)
    m = torch.where(mc == 0, 0.0, torch.where(mc == 127, float("nan"), torch.where((c & 0x80) != 0, -m, m)))
    v = ((vc << 20) + (bv << 23)).view(torch.float32)
    return m, torch.where(vc == 0, 0.0, torch.where(vc == 255, float("inf"), v))


def plain_norm(grads):
    return grads.double().square().sum().sqrt().float()


def plain_step(s, m, v):
    """One step of torch.optim.AdamW on the flat buffers, from the old moments (f32, one row a block); -> the new moments."""
    t, case = s["step"], s["case"]
    b1, b2 = BETAS
    g = s["grads"].float().view(-1, BLOCK)
    norm = None
    if case["max_norm"]:
        norm = plain_norm(s["grads"])
        g = g * (case["max_norm"] / (norm.double() + 1e-6)).clamp(max=1.0).float()
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * (1 - b2) * g
    w = (s["params"].float() if s["masters"] is None else s["masters"]).view(-1, BLOCK)
    lr = s["lr_column"]
    w = w * (1 - lr * s["decay_column"]).float()
    w = w - (lr / (1 - b1 ** t)).float() * (m / (v.sqrt() * (1 - b2 ** t) ** -0.5 + s["eps"]))
    if s["masters"] is not None:
        s["masters"].copy_(w.view(-1))
    s["params"].copy_(w.view(-1))
    return m, v, norm


def run(s):
    op = s["case"]["op"]
    if op == "norm":
        if own:
            from gs_icp_slam_amd.optim import grad_norm
            return {"norm": grad_norm(s["grad_list"])}
        return {"norm": plain_norm(s["grads"])}
    s["step"] += 1
    max_norm = s["case"]["max_norm"] or None
    if op == "adamw":
        if own:
            from gs_icp_slam_amd.optim import adamw_step
            norm = adamw_step(s["param_list"], s["grad_list"], s["exp_avg_list"], s["exp_avg_sq_list"], lr=s["lr"], betas=BETAS, eps=s["eps"],
                              weight_decay=s["weight_decay"], step=s["step"], masters=s["master_list"], max_norm=max_norm)
        else:
            m, v, norm = plain_step(s, s["exp_avg"].view(-1, BLOCK), s["exp_avg_sq"].view(-1, BLOCK))
            s["exp_avg"].copy_(m.view(-1))
            s["exp_avg_sq"].copy_(v.view(-1))
        return {"params": s["params"], "masters": s["masters"], "exp_avg": s["exp_avg"], "exp_avg_sq": s["exp_avg_sq"], "norm": norm}
    if own:
        from gs_icp_slam_amd.optim import adamw_step_8bit, decode_moments
        norm = adamw_step_8bit(s["param_list"], s["grad_list"], s["moment_list"], s["block_exp_list"], lr=s["lr"], betas=BETAS, eps=s["eps"],
                               weight_decay=s["weight_decay"], step=s["step"], seed=s["seed"], masters=s["master_list"], max_norm=max_norm)
        # the buffer as a whole is one tensor of whole blocks; the codes' values have four significant bits: bfloat16 holds them as they are
        (m,), (v,) = decode_moments([s["moments"]], [s["block_exps"]], dtype=torch.bfloat16)
    else:
        m, v, norm = plain_step(s, *decode(s["moments"], s["block_exps"]))
        s["moments"], s["block_exps"] = encode(m, v, *random_words(s, s["step"]))
        m, v = (x.bfloat16().view(-1) for x in decode(s["moments"], s["block_exps"]))
    return {"params": s["params"], "masters": s["masters"], "exp_avg": m, "exp_avg_sq": v, "norm": norm}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def value_of(code, base):
    """What a code stands for, by the definition: (1 + mantissa / 8) * 2^(exponent)."""
    c = code.double()
    return torch.where(code > 0, torch.ldexp(1 + torch.remainder(c, 8) / 8, torch.floor(c / 8) + base.double() - 127), torch.zeros_like(c))


def code_of(x, base, u):
    """x > 0 rounded to a code: up with the probability of its distance to the code below, as u (in (0, 1)) says."""
    f, e = torch.frexp(x)
    return ((e + 126 - base) * 8 + torch.floor((2 * f - 1) * 8 + u)).long()


def exact(case, seed):
    s = prepare(case, seed)
    g = s["grads"].double()
    norm = torch.linalg.vector_norm(g)
    if case["op"] == "norm":
        return {"norm": norm}
    b1, b2 = BETAS
    t = s["step"] + 1
    if case["op"] == "adamw8":
        codes, exps = s["moments"].long().view(-1, BLOCK) & 0xFFFF, s["block_exps"].long().view(-1, 1) & 0xFFFF
        m = value_of(codes % 128, exps % 256) * (1 - 2 * (codes // 128 % 2))
        v = value_of(codes // 256, exps // 256)
    else:
        m, v = s["exp_avg"].double().view(-1, BLOCK), s["exp_avg_sq"].double().view(-1, BLOCK)
    if case["max_norm"]:
        g = g * min(1.0, case["max_norm"] / (float(norm) + 1e-6))
    g = g.view(-1, BLOCK)
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    w = (s["params"] if s["masters"] is None else s["masters"]).double().view(-1, BLOCK)
    lr = s["lr_column"]
    w = w - lr * s["decay_column"] * w - lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + s["eps"])
    if case["op"] == "adamw8":
        r = (mix(s["octet"] ^ mix((s["seed"] + t * G1 + s["place"] * G2) & M32)).unsqueeze(2) * torch.tensor(LANE, device=w.device) & M32).view(-1, BLOCK)
        um, uv = (r % 65536).double(), (r // 65536).double()
        a = m.abs()
        bm = (torch.frexp(a.amax(1, keepdim=True))[1] + 126 - 14).clamp_min(1)
        bv = (torch.frexp(v.amax(1, keepdim=True))[1] + 126 - 30).clamp_min(1)
        low = value_of(torch.ones_like(bm), bm)
        mc = torch.where(a < low, (a > low * (um + 0.5) / 65536).long(), code_of(a, bm, (um + 0.5) / 65536))
        vc = torch.where(v > 0, code_of(v, bv, (uv + 0.5) / 65536).clamp_min(1), 0)
        m, v = value_of(mc, bm) * torch.sign(m), value_of(vc, bv)
    return {"params": w.view(-1), "masters": None if s["masters"] is None else w.view(-1), "exp_avg": m.view(-1), "exp_avg_sq": v.view(-1),
            "norm": norm if case["max_norm"] else None}
