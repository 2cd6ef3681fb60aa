"""The optimizer's operators as measured calls: an AdamW step over many tensors with its moments in 32 or in 8 bits, and the
clipping of gradients by their global norm.

``own = False`` computes them in elementary torch operations over flat buffers; ``own = True`` calls remixfusion_amd.optim.
Parameters, gradients and moments of a case lie in flat buffers, each tensor at a multiple of 256 elements (a tensor of an
allocator of its own starts at a multiple of 512 bytes as well); what lies between two tensors is zero and stays zero.

8-bit moments: blocks of 256 elements of a tensor share an exponent E (an int8: E of exp_avg, E / 2 of exp_avg_sq, whose range is
twice as wide); an element is a small float under it.
  exp_avg    sign, 4 bits f, 3 bits n     value  n 2^(E-17) (f = 0)   (8 + n) 2^(E-18+f)
  exp_avg_sq       5 bits f, 3 bits n     value  n 2^(E-33) (f = 0)   (8 + n) 2^(E-34+f)
E is the exponent of the block's largest magnitude, one more where its significand is 1.875 or above, and for exp_avg_sq one more
where that is odd.  The moment is rounded to 20
bits below the format's last place, then up with the probability of the rest, by 16 bits of a hash of (seed, step, tensor, block,
element); a second moment that is not zero stays at least one unit of the last place."""
import math
import random

import torch

own = False

BLOCK = 256
SEED = 1234                      # of the hash that the 8-bit moments are rounded with
DECODER = [(32, 81), (16, 32), (32, 66), (3, 32)]                                                        # the field's decoder
POSE_MLP = [(256, 7), (256,), (256, 256), (256,), (256, 256), (256,), (6, 256), (6,)]                  # the pose network
TABLES = {"office0": 1640944, "scene0000": 10269056, "cafeteria": 41549648}                             # hash tables, floats


def _case(name, op, shapes, **kw):
    c = {"name": name, "op": op, "shapes": shapes, "tensors": 0, "total": 0, "dtype": "float32", "master": False, "clip": False,
         "norm": "2", "lr": 1e-3, "beta1": 0.9, "beta2": 0.99, "eps": 1e-8, "weight_decay": 1e-2, "step": 40}
    c.update(kw)
    return c


def listed():
    return [
        # a decoder by itself: 5 312 parameters, what a step costs when latency is all there is
        _case("step32_decoder", "step32", "decoder", lr=0.01, weight_decay=1e-6),
        # the pose network's eight tensors, clipped: two small passes that depend on each other
        _case("step32_pose_mlp_clip", "step32", "pose_mlp", clip=True, lr=5e-4, eps=1e-15, weight_decay=1e-6),
        # the map optimizer at the smallest scene's table
        _case("step32_office0", "step32", "office0", lr=0.01, eps=1e-15),
        # ... and at the largest scene's: 1.2 GB of traffic
        _case("step32_cafeteria", "step32", "cafeteria", lr=0.01, eps=1e-15),
        # ragged tensors of a 16-bit model with fp32 master weights, clipped
        _case("step32_bf16_master_clip", "step32", "spread", tensors=15, total=8_000_003, dtype="bfloat16", master=True, clip=True, beta2=0.95),
        # 8-bit moments where little is to be gained: the pose network
        _case("step8_pose_mlp", "step8", "pose_mlp", lr=5e-4, weight_decay=1e-6),
        # a middle-sized table, clipped
        _case("step8_scene0000_clip", "step8", "scene0000", clip=True, lr=0.01, eps=1e-15),
        # the largest table, whose step is what moves the most bytes
        _case("step8_cafeteria", "step8", "cafeteria", lr=0.01, eps=1e-15),
        # ragged half-precision tensors without a master copy
        _case("step8_fp16", "step8", "spread", tensors=13, total=3_000_001, dtype="float16", beta2=0.999),
        # clipping by itself: below the limit (most steps of a run: nothing is written), small
        _case("clip_pose_mlp_under", "clip", "pose_mlp"),
        # above the limit: new gradients come in with each pass and are rewritten
        _case("clip_office0_over", "clip", "office0", clip=True),
        # the largest set of gradients, read once
        _case("clip_cafeteria_under", "clip", "cafeteria"),
    ]


def draw(rng):
    op = rng.choice(["step32", "step8", "clip"])
    dtype = rng.choice(["float32", "float32", "bfloat16", "float16"])
    total = int(math.exp(rng.uniform(math.log(1000), math.log(4.0e7))))
    c = _case("", op, "spread", tensors=rng.randint(1, 15), total=total, dtype=dtype, clip=rng.random() < 0.5)
    del c["name"]
    c["master"] = dtype != "float32" and op != "clip" and rng.random() < 0.5
    c["norm"] = rng.choice(["2", "2", "inf"]) if op == "clip" else "2"
    c["lr"], c["beta2"] = 10.0 ** rng.uniform(-4, -2), rng.choice([0.95, 0.99, 0.999])
    c["eps"], c["weight_decay"], c["step"] = rng.choice([1e-15, 1e-8]), rng.choice([0.0, 1e-6, 1e-2, 0.1]), rng.randint(1, 2000)
    return c


def _shapes(case):
    if case["shapes"] == "decoder":
        return DECODER
    if case["shapes"] == "pose_mlp":
        return POSE_MLP
    if case["shapes"] in TABLES:
        return DECODER + [(TABLES[case["shapes"]],)]
    r = random.Random(case["total"])                     # ragged: sizes over three orders of magnitude, few of them even
    w = [10.0 ** r.uniform(-3, 0) for _ in range(case["tensors"])]
    return [(max(1, int(case["total"] * x / sum(w))),) for x in w]


def _count(case):
    return sum(math.prod(s) for s in _shapes(case))


def work(case):
    n, size = _count(case), 4 if case["dtype"] == "float32" else 2
    if case["op"] == "clip":
        return {"bytes": n * size * (2 if case["clip"] else 1), "flops": 2 * n}
    weights = 8 + size if case["master"] else 2 * size                      # a master copy is read and written, its parameter only written
    moments = 16 if case["op"] == "step32" else 4 + 4 / BLOCK + 8           # 8 bits: the values are read back in 32
    return {"bytes": n * (weights + size + moments), "flops": n * (14 + (2 if case["clip"] else 0))}


def _views(flat, s):
    return [flat[o:o + n].view(shape) for o, n, shape in s["places"]]


def _exponents(largest, unit):
    """the int8 of blocks whose largest magnitude is given (fp64): E in units of 1 or 2"""
    f, k = torch.frexp(largest)
    e = k - 1 + (f >= 0.9375).to(k.dtype)
    return torch.where(largest > 0, (e + unit - 1) // unit, torch.full_like(k, -127)).clamp(-127, 127)


def _encode_nearest(x, floor, top):
    """codes (no sign) and exponents of |x| [blocks, 256], to nearest: how the inputs of a case are made"""
    y = x.abs().double()
    unit = 1 if floor == -14 else 2
    E = _exponents(y.amax(1), unit)
    y = y * torch.exp2(-unit * E.double())[:, None]
    _, k = torch.frexp(y)
    e = torch.where(y > 0, k - 1, torch.full_like(k, floor)).clamp(min=floor)
    n = torch.round(y * torch.exp2(3.0 - e.double()))
    return (n + 8 * (e - floor)).clamp(max=top).to(torch.uint8), E.to(torch.int8)


def prepare(case, seed):
    shapes = _shapes(case)
    dev, dtype = torch.device("cuda"), getattr(torch, case["dtype"])
    places, at = [], 0
    for shape in shapes:
        n = math.prod(shape)
        places.append((at, n, shape))
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    gen = torch.Generator(device=dev).manual_seed(seed)
    live = torch.zeros(at, device=dev)
    for o, n, _ in places:
        live[o:o + n] = 1.0

    def normal():
        return torch.randn(at, device=dev, generator=gen) * live

    # magnitudes over a few orders, and a third of the elements (a table's entries that no sample met) without any gradient
    size = 1e-3 * torch.exp(1.5 * normal())
    met = (torch.rand(at, device=dev, generator=gen) > 0.33).float()
    s = {"case": case, "places": places, "step": case["step"]}
    s["G"] = (normal() * size * met).to(dtype)
    if case["op"] == "clip":
        s["G0"] = s["G"].clone() if case["clip"] else None
    else:
        master = 0.1 * normal()
        s["P"] = master.to(dtype)
        s["W"] = master if case["master"] else None
        m, v = 0.3 * normal() * size, live * size * size * (0.2 + torch.rand(at, device=dev, generator=gen))
        if case["op"] == "step32":
            s["M"], s["V"] = m, v
        else:
            cm, em = _encode_nearest(m.view(-1, BLOCK), -14, 127)
            cv, ev = _encode_nearest(v.view(-1, BLOCK), -30, 255)
            s["M"] = (cm + 128 * (m.view(-1, BLOCK) < 0).to(torch.uint8)).view(-1)
            s["V"], s["E"] = cv.view(-1), torch.stack([em, ev])
            blocks = [(n + BLOCK - 1) // BLOCK for _, n, _ in places]
            s["block_tensor"] = torch.repeat_interleave(torch.arange(len(blocks), device=dev), torch.tensor(blocks, device=dev))
            first = torch.tensor([o // BLOCK for o, _, _ in places], device=dev)
            s["block"] = torch.arange(at // BLOCK, device=dev) - first[s["block_tensor"]]
    norm = float(s["G"].double().abs().max() if case["norm"] == "inf" else s["G"].double().square().sum().sqrt())
    s["limit"] = norm * (0.7 if case["clip"] else 4.0)
    s["grads"] = _views(s["G"], s)
    if case["op"] != "clip":
        s["params"] = _views(s["P"], s)
    if own:
        _own_handle(s)
    return s


def _own_handle(s):
    """what a user's program keeps: parameters with their gradients, and the optimizer with its state"""
    case = s["case"]
    s["leaves"] = [torch.nn.Parameter(t) for t in s.get("params", [torch.empty_like(g) for g in s["grads"]])]
    for p, g in zip(s["leaves"], s["grads"]):
        p.grad = g
    if case["op"] == "clip":
        return
    from remixfusion_amd.optim import AdamW
    opt = AdamW(s["leaves"], lr=case["lr"], betas=(case["beta1"], case["beta2"]), eps=case["eps"], weight_decay=case["weight_decay"],
                state_bits=32 if case["op"] == "step32" else 8, master_weights=case["master"],
                max_grad_norm=s["limit"] if case["clip"] else None, seed=SEED)
    state, m, v = {}, _views(s["M"], s), _views(s["V"], s)
    for i, (o, n, shape) in enumerate(s["places"]):
        state[i] = {"step": torch.tensor(float(s["step"])), "exp_avg": m[i], "exp_avg_sq": v[i]}
        if case["op"] == "step8":
            state[i]["exponents"] = s["E"][:, o // BLOCK:(o + n + BLOCK - 1) // BLOCK].contiguous()
        if case["master"]:
            state[i]["master"] = s["W"][o:o + n].view(shape)
    opt.load_state_dict({"state": state, "param_groups": opt.state_dict()["param_groups"]})
    s["opt"] = opt


def run(s):
    case = s["case"]
    if case["op"] == "clip":
        if case["clip"]:
            s["G"].copy_(s["G0"])                    # stands for the backward pass, which brings gradients that are not clipped yet
        if own:
            from remixfusion_amd.optim import clip_grad_norm_
            norm = clip_grad_norm_(s["leaves"], s["limit"], norm_type=float(case["norm"]))
        else:
            norm = _norm(s)
            s["G"].copy_((s["G"].float() * _factor(s, norm).float()).to(s["G"].dtype))
            norm = norm.float()
        return {"norm": norm, "grads": s["grads"]}
    if not own:
        return _plain_step(s)
    opt = s["opt"]
    opt.step()
    out = {"params": s["params"]}
    if case["op"] == "step32":
        states = [opt.state[p] for p in s["leaves"]]
        out["exp_avg"], out["exp_avg_sq"] = [t["exp_avg"] for t in states], [t["exp_avg_sq"] for t in states]
    else:
        out["exp_avg"], out["exp_avg_sq"] = opt.moments()            # held in 8 bits: the values they stand for
    if case["master"]:
        out["master"] = [opt.state[p]["master"] for p in s["leaves"]]
    if case["clip"]:
        out["norm"] = opt.grad_norm
    return out


# ---- the plain form ------------------------------------------------------------------------------------------------------
def _norm(s):
    """global norm of the gradients, fp64: a long sum, and a factor in front of values that are rounded to 8 bits"""
    g = s["G"].double()
    return g.abs().max() if s["case"]["norm"] == "inf" else g.square().sum().sqrt()


def _factor(s, norm):
    return (s["limit"] / (norm + 1e-6)).clamp(max=1.0)


def _plain_step(s):
    case = s["case"]
    s["step"] += 1
    b1, b2, k = case["beta1"], case["beta2"], s["step"]
    norm = _norm(s) if case["clip"] else None
    if case["op"] == "step32":
        g = s["G"].float()
        if case["clip"]:
            g = g * _factor(s, norm).float()
        m = s["M"].copy_(s["M"] * b1 + g * (1 - b1))
        v = s["V"].copy_(s["V"] * b2 + g * g * (1 - b2))
        values = m, v
    else:
        g = s["G"].double()
        if case["clip"]:
            g = g * _factor(s, norm)
        e1, e2 = s["E"][0].double(), 2 * s["E"][1].double()
        m = _decode((s["M"] & 127), e1 - 17) * (1.0 - 2.0 * (s["M"] >> 7).double()) * b1 + g * (1 - b1)
        v = _decode(s["V"], e2 - 33) * b2 + g * g * (1 - b2)
        bits = _bits(s, k)
        code, e1, dm = _round(m.abs().view(-1, BLOCK), -14, 127, bits & 0xffff)
        s["M"].copy_((code + 128 * (m < 0).to(torch.int64)).to(torch.uint8))
        dm = dm * torch.where(m < 0, -1.0, 1.0)
        code, e2, dv = _round(v.view(-1, BLOCK), -30, 255, bits >> 16, True)
        s["V"].copy_(code.to(torch.uint8))
        s["E"].copy_(torch.stack([e1, e2]).to(torch.int8))
        values = dm.float(), dv.float()
        m, v = m.float(), v.float()
    p = s["W"] if case["master"] else s["P"].float()
    denominator = v.sqrt() / math.sqrt(1 - b2 ** k) + case["eps"]
    p = p * (1 - case["lr"] * case["weight_decay"]) - (m / denominator) * (case["lr"] / (1 - b1 ** k))
    s["P"].copy_(p.to(s["P"].dtype))
    out = {"params": s["params"], "exp_avg": _views(values[0], s), "exp_avg_sq": _views(values[1], s)}
    if case["master"]:
        out["master"] = _views(s["W"].copy_(p), s)
    if case["clip"]:
        out["norm"] = norm.float()
    return out


def _decode(code, unit):
    f, n = (code >> 3).to(torch.int64), (code & 7).double()
    scale = torch.exp2(unit)[:, None]
    value = torch.where(f == 0, n, (n + 8.0) * torch.exp2((f - 1).double()))
    return (value.view(-1, BLOCK) * scale).view(-1)


def _mix(x):
    """two-multiply mixer of 32-bit integers, held in int64"""
    x = ((x ^ (x >> 16)) * 0x7feb352d) & 0xffffffff
    x = ((x ^ (x >> 15)) * 0x846ca68b) & 0xffffffff
    return x ^ (x >> 16)


def _bits(s, step):
    key = _mix(torch.full_like(s["block_tensor"], SEED))
    key = _mix((key + step) & 0xffffffff)
    key = _mix((key + s["block_tensor"]) & 0xffffffff)
    block = _mix((key + s["block"]) & 0xffffffff)
    lane = (torch.arange(BLOCK, device=block.device) * 0x9e3779b9) & 0xffffffff
    return _mix((block[:, None] + lane[None, :]) & 0xffffffff)


def _round(y, floor, top, bits, keep=False):
    """codes, exponents and values of y >= 0 [blocks, 256]; the smallest normal's exponent under E is `floor`"""
    largest = y.amax(1)
    unit = 1 if floor == -14 else 2
    E = _exponents(largest, unit)
    scale = torch.exp2(unit * E.double())[:, None]
    y = y / scale
    _, k = torch.frexp(y)
    e = torch.where(y > 0, k - 1, torch.full_like(k, floor)).clamp(min=floor)
    t = torch.round(y * torch.exp2(23.0 - e.double()))
    n = torch.floor((t + (bits * 16 + 8)) * 2.0 ** -20).to(torch.int64)
    code = (n + 8 * (e - floor)).clamp(max=top)
    if keep:
        code = torch.where(y > 0, code.clamp(min=1), code)
    f, n = code >> 3, (code & 7).double()
    value = torch.where(f == 0, n, (n + 8.0) * torch.exp2((f - 1).double())) * 2.0 ** (floor - 3) * scale
    return code.view(-1), E, value.view(-1)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    G = [g.double() for g in s["grads"]]
    if case["norm"] == "inf":
        norm = torch.stack([g.abs().max() for g in G]).max()
    else:
        norm = torch.sqrt(sum(torch.dot(g.reshape(-1), g.reshape(-1)) for g in G))
    c = min(1.0, s["limit"] / (float(norm) + 1e-6))
    if case["op"] == "clip":
        return {"norm": norm, "grads": [g * c for g in G]}
    if not case["clip"]:
        c = 1.0
    k, b1, b2 = case["step"] + 1, case["beta1"], case["beta2"]
    out = {"params": [], "exp_avg": [], "exp_avg_sq": []}
    if case["master"]:
        out["master"] = []
    for i, (o, n, shape) in enumerate(s["places"]):
        g = G[i].reshape(-1) * c
        p = (s["W"] if case["master"] else s["P"])[o:o + n].double()
        m, v = s["M"][o:o + n], s["V"][o:o + n]
        if case["op"] == "step8":
            E = s["E"][:, o // BLOCK:(o + n + BLOCK - 1) // BLOCK].double().repeat_interleave(BLOCK, 1)[:, :n]
            small = torch.arange(256, device=m.device)
            table = torch.where(small < 8, small.double(), (small % 8 + 8).double() * 2.0 ** (small // 8 - 1).double())
            sign = torch.where(m >= 128, -1.0, 1.0).double()
            m, v = table[(m % 128).long()] * sign * 2.0 ** (E[0] - 17), table[v.long()] * 2.0 ** (2 * E[1] - 33)
        m = b1 * m.double() + (1 - b1) * g
        v = b2 * v.double() + (1 - b2) * g ** 2
        p = (1 - case["lr"] * case["weight_decay"]) * p - case["lr"] / (1 - b1 ** k) * m / ((v / (1 - b2 ** k)).sqrt() + case["eps"])
        if case["op"] == "step8":
            r = _exact_bits(k, i, n, m.device)
            m, v = m.sign() * _exact_round(m.abs(), r % 65536, 15), _exact_round(v, r // 65536, 31)
        for key, x in (("params", p), ("exp_avg", m), ("exp_avg_sq", v)) + ((("master", p),) if case["master"] else ()):
            out[key].append(x.reshape(shape))
    if case["clip"]:
        out["norm"] = norm
    return out


def _exact_bits(step, index, n, device):
    import numpy as np

    def mix(x):
        x = x.astype(np.uint32)
        with np.errstate(over="ignore"):
            x ^= x >> np.uint32(16)
            x *= np.uint32(0x7feb352d)
            x ^= x >> np.uint32(15)
            x *= np.uint32(0x846ca68b)
            return x ^ (x >> np.uint32(16))

    key = np.array([SEED], np.uint64)
    for more in (step, index):
        key = (mix(key).astype(np.uint64) + np.uint64(more)) & np.uint64(0xffffffff)
    key = mix(key).astype(np.uint64)
    blocks = mix((key + np.arange((n + BLOCK - 1) // BLOCK, dtype=np.uint64)) & np.uint64(0xffffffff))
    lane = (np.arange(BLOCK, dtype=np.uint64) * np.uint64(0x9e3779b9) & np.uint64(0xffffffff)).astype(np.uint32)
    r = mix((blocks[:, None] + lane[None, :]).reshape(-1))[:n]
    return torch.from_numpy(r.astype(np.int64)).to(device)


def _exact_round(y, r, octaves):
    """y >= 0 as the format of so many octaves under each block's exponent holds it; r: 16 random bits"""
    n = y.numel()
    y = torch.nn.functional.pad(y, (0, -n % BLOCK)).view(-1, BLOCK)
    r = torch.nn.functional.pad(r, (0, -n % BLOCK)).view(-1, BLOCK).double()
    top = y.max(dim=1, keepdim=True).values
    E = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    E = torch.where(2.0 ** E > top, E - 1, torch.where(2.0 ** (E + 1) <= top, E + 1, E))
    E = torch.where(top >= 1.875 * 2.0 ** E, E + 1, E)
    E = torch.where(E % 2 == 1, E + 1, E) if octaves == 31 else E
    E = torch.where(top > 0, E.clamp(-127, 127) if octaves == 15 else E.clamp(-254, 254), torch.zeros_like(E))
    k = torch.frexp(y).exponent.double() - 1                                # unit of the last place of each element's octave
    unit = 2.0 ** (torch.maximum(k, E - octaves + 1) - 3)
    t = torch.round(y / unit * 2.0 ** 20)
    z = torch.floor((t + 16 * r + 8) / 2.0 ** 20) * unit
    z = torch.minimum(z, 1.875 * 2.0 ** E)
    least = 2.0 ** (E - octaves - 2)
    z = torch.maximum(z, least) if octaves == 31 else z
    return torch.where(y > 0, z, torch.zeros_like(z)).view(-1)[:n]
