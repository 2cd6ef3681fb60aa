"""remixfusion_amd.optim.AdamW (rfx_adamw_step, rfx_adamw_moments) and clip_grad_norm_ (rfx_grad_norm, rfx_grad_scale) against a plain
numpy implementation in 64 bits.

Tolerances.  u = 2^-24 is half a unit of fp32's last place.  32-bit moments: g c (1), the two factors (1 each), two roundings
of the sum: at most 4 u (|b1 m| + |c1 g|), and 5 u for v with its square.  The parameter: its own rounding (u |p|, or eps/2 of its
type, which a master copy does not see), and of the update: m's error over the denominator, and m / d with sqrt, 1/sqrt(1-b2^k), eps, the fma,
the division, the product with lr/(1-b1^k) and v's error halved by the root: under 16 u |update|.  8-bit moments are formed in fp64 on both sides: their codes and exponents have to be EQUAL
(a border would have to lie within 1e-15 of a value), and the update gets the rounding of m and v to fp32 on top, inside the same 16 u."""
import copy
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_eps(dtype):
    return torch.finfo(dtype).eps / 2


# ---- the oracle -----------------------------------------------------------------------------------------------------------
def mix(x):
    x = np.asarray(x, dtype=np.uint64) & 0xffffffff
    for shift, mul in ((16, 0x7feb352d), (15, 0x846ca68b)):
        x = ((x ^ (x >> np.uint64(shift))) * np.uint64(mul)) & np.uint64(0xffffffff)
    return x ^ (x >> np.uint64(16))


def noise(seed, step, index, n, first=0):
    """the 32 bits of elements [first, first + n) of a tensor; first: a multiple of 256"""
    key = mix(mix(mix(seed) + np.uint64(step)) + np.uint64(index))
    i = np.arange(first, first + n, dtype=np.uint64)
    run = mix(key + (i >> np.uint64(8)))
    return mix(run + (i & np.uint64(255)) * np.uint64(0x9e3779b9))


def runs(x):
    n = len(x)
    return np.concatenate([x, np.zeros(-n % 256, x.dtype)]).reshape(-1, 256)


def encode(x, bits16, octaves):
    """codes (with a sign bit if octaves is 15), exponents"""
    top, floor = 8 * octaves + 7, 2 - octaves - 1                       # the smallest normal octave under E
    y = runs(np.abs(x))
    big = y.max(1)
    finite = np.isfinite(big)
    big = np.where(finite, big, 1.0)
    f, k = np.frexp(big)
    E = np.where(big > 0, k - 1 + (2 * f >= 1.875), -127)
    unit = 1 if octaves == 15 else 2                                    # exp_avg_sq: even exponents, halved
    h = np.where(big > 0, np.clip(-(-E // unit), -127, 127), -127)
    E = h * unit
    y = np.where(finite[:, None], y, 0.0) * 2.0 ** -E[:, None].astype(float)
    _, k = np.frexp(y)
    e = np.where(y > 0, np.maximum(k - 1, floor), floor)
    t = np.rint(y * 2.0 ** (23.0 - e))
    n = np.floor((t + runs(bits16).astype(float) * 16 + 8) / 2.0 ** 20)
    code = np.minimum(n + 8 * (e - floor), top)
    if octaves == 31:
        code = np.where(y > 0, np.maximum(code, 1), code)
    code = np.where(finite[:, None], code, 0).astype(np.uint8).reshape(-1)[:len(x)]
    return code, np.where(finite, h, -128).astype(np.int8)


def decode(code, E, octaves):
    c = code.astype(int) & (8 * octaves + 7)
    f, n = c >> 3, c & 7
    lost = np.repeat(E == -128, 256)[:len(code)]
    E = np.repeat(E.astype(float) * (1 if octaves == 15 else 2), 256)[:len(code)]
    x = np.where(f == 0, n * 2.0 ** (E - octaves - 2), (8 + n) * 2.0 ** (E - octaves - 3 + f))
    x = np.where(lost, np.nan, x)
    return np.where(code >= 128, -x, x) if octaves == 15 else x


class Ref:
    """one tensor, everything in fp64; p as the kernel was given it"""

    def __init__(self, p, bits=32, index=0, seed=0):
        self.p, self.bits, self.index, self.seed, self.k = p.astype(np.float64), bits, index, seed, 0
        self.m, self.v = np.zeros_like(self.p), np.zeros_like(self.p)
        self.cm, self.cv = np.zeros(len(p), np.uint8), np.zeros(len(p), np.uint8)
        self.e1 = self.e2 = np.full(-(-len(p) // 256), -127, np.int8)

    def step(self, g, lr, betas, eps, weight_decay, c=1.0, half=U, first=0):
        """-> error bounds of (p, m, v); first: place of element 0 in its tensor"""
        self.k += 1
        b1, b2 = betas
        g = g.astype(np.float64) * c
        with np.errstate(all="ignore"):
            bm, bv = b1 * self.m, b2 * self.v
            m, v = bm + (1 - b1) * g, bv + (1 - b2) * g * g
            tm, tv = 4 * U * (np.abs(bm) + np.abs((1 - b1) * g)), 5 * U * v + 2.0 ** -149
            d = np.sqrt(v) / math.sqrt(1 - b2 ** self.k) + eps
            size = lr / (1 - b1 ** self.k)
            up = size * m / d
            p = self.p - lr * weight_decay * self.p - up
            tp = half * np.abs(p) + U * np.abs(self.p) + 16 * U * np.abs(up) + size * tm / d + 2.0 ** -149
            if half > 2.0 ** -20:
                tp = tp * 1.0001 + (2.0 ** -25 if half == 2.0 ** -11 else 0)      # fp16's subnormals: half a unit of 2^-24
        self.p, self.m, self.v = p, m, v
        if self.bits == 8:
            r = noise(self.seed, self.k, self.index, len(p), first)
            self.cm, self.e1 = encode(m, r & np.uint64(0xffff), 15)
            self.cm |= ((m < 0) * 128).astype(np.uint8)
            self.cv, self.e2 = encode(v, r >> np.uint64(16), 31)
            self.m, self.v = decode(self.cm, self.e1, 15), decode(self.cv, self.e2, 31)
            tm = tv = np.zeros_like(p)
        return tp, tm, tv


def near(got, want, tol, what):
    got = got.detach().double().cpu().numpy().reshape(-1)
    want, tol = np.asarray(want, np.float64).reshape(-1), np.broadcast_to(np.asarray(tol, np.float64).reshape(-1), want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), (what, "NaN")
    ok = np.isnan(want) | (got == want) | (np.abs(got - want) <= tol)
    if not ok.all():
        i = int(np.argmax(~ok))
        raise AssertionError(f"{what}: element {i} of {len(want)} ({int((~ok).sum())} off): {got[i]!r} for {want[i]!r}, tolerance {tol[i]!r}")


def magnitudes(n, gen, zeros=0.3):
    """gradients over some orders of magnitude, part of them zero"""
    g = torch.randn(n, device="cuda", generator=gen) * torch.exp(2.0 * torch.randn(n, device="cuda", generator=gen)) * 1e-2
    return g * (torch.rand(n, device="cuda", generator=gen) >= zeros)


SIZES = [1, 2, 3, 5, 64, 255, 256, 257, 511, 1023, 4095, 4096, 4097, 8191, 12289, 70001]
SETTINGS = [dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-15, weight_decay=1e-6), dict(lr=3e-3, betas=(0.8, 0.999), eps=1e-8, weight_decay=0.1)]


def _check_code(st, ref, what):
    assert np.array_equal(st["exponents"].cpu().numpy(), np.stack([ref.e1, ref.e2])), (what, "exponents")
    assert np.array_equal(st["exp_avg_sq"].cpu().numpy().reshape(-1), ref.cv), (what, "exp_avg_sq")
    near(torch.from_numpy(decode(st["exp_avg"].cpu().numpy().reshape(-1), ref.e1, 15)), ref.m, 0.0, (what, "exp_avg"))


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("bits", [32, 8])
def test_steps_match_64_bits(bits, dtype, master, offset):
    """sizes around every border of the kernels, two groups, three steps; offset 1: parameters and gradients that no vector load fits"""
    from remixfusion_amd.optim import AdamW
    if master and dtype == "f32":
        pytest.skip("an fp32 parameter is its own master copy")
    T = DTYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(11)
    buf = [torch.randn(n + offset, device="cuda", generator=gen).mul(0.3).to(T) for n in SIZES]
    guard = [b.clone() for b in buf]
    ps = [torch.nn.Parameter(b[offset:]) for b in buf]
    half = len(ps) // 2
    opt = AdamW([dict(params=ps[:half], **SETTINGS[0]), dict(params=ps[half:], maximize=True, **SETTINGS[1])],
                state_bits=bits, master_weights=master, seed=99)
    refs = [Ref(p.detach().float().cpu().numpy(), bits, i, 99) for i, p in enumerate(ps)]
    for it in range(3):
        for p in ps:
            g = torch.empty(p.numel() + offset, device="cuda", dtype=T)
            g[offset:] = magnitudes(p.numel(), gen).to(T)
            p.grad = g[offset:]
        opt.step()
        for i, (p, ref) in enumerate(zip(ps, refs)):
            s, sign = SETTINGS[i >= half], 1.0 if i < half else -1.0
            tp, tm, tv = ref.step(p.grad.float().cpu().numpy(), **s, c=sign, half=U if master else half_eps(T))
            st, what = opt.state[p], (it, p.numel())
            assert float(st["step"]) == it + 1
            if bits == 8:
                _check_code(st, ref, what)
            else:
                near(st["exp_avg"], ref.m, tm, (what, "m"))
                near(st["exp_avg_sq"], ref.v, tv, (what, "v"))
                ref.m, ref.v = (st[k].double().cpu().numpy() for k in ("exp_avg", "exp_avg_sq"))
            if master:
                near(st["master"], ref.p, tp, (what, "master"))
                assert torch.equal(p.detach(), st["master"].to(T)), what               # one rounding, to nearest
                ref.p = st["master"].double().cpu().numpy()
            else:
                near(p, ref.p, tp, (what, "p"))
                ref.p = p.detach().double().cpu().numpy()                            # the next step starts from what is there
    for b, b0, p in zip(buf, guard, ps):
        assert torch.equal(b[:offset], b0[:offset])
    avg, avg_sq = opt.moments()
    for p, ref, a, b in zip(ps, refs, avg, avg_sq):
        near(a, ref.m, 0.0, "moments"); near(b, ref.v, U * np.abs(ref.v) + 2.0 ** -149, "moments")


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_equal_one_by_one(bits):
    """310 tensors in eleven groups go through several launches; each alone gives the same bits"""
    from remixfusion_amd.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(5)
    sizes = [int(x) for x in np.random.default_rng(3).integers(0, 700, 310)]          # some without any element
    init, grads = ([torch.randn(n, device="cuda", generator=gen) for n in sizes] for _ in range(2))
    ps = [torch.nn.Parameter(t.clone()) for t in init]
    groups = [dict(params=ps[k::11], lr=1e-3 * (k + 1)) for k in range(11)]
    opt = AdamW(groups, state_bits=bits, seed=4)
    order = [i for k in range(11) for i in range(310)[k::11]]
    for p, g in zip(ps, grads):
        p.grad = g
    for _ in range(2):
        opt.step()
    for place, i in enumerate(order):
        if i % 7 and sizes[i]:
            continue
        fill = [torch.nn.Parameter(torch.zeros(0, device="cuda")) for _ in range(place)]       # the same place in its optimizer
        q = torch.nn.Parameter(init[i].clone())
        one = AdamW(fill + [q], lr=1e-3 * (i % 11 + 1), state_bits=bits, seed=4)
        q.grad = grads[i]
        for _ in range(2):
            one.step()
        assert torch.equal(q, ps[i]) and float(opt.state[ps[i]]["step"]) == 2.0
        for key in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(one.state[q][key], opt.state[ps[i]][key])


@pytest.mark.parametrize("bits,dtype,master", [(32, "f32", False), (8, "f32", False), (32, "bf16", True), (8, "f16", False), (8, "bf16", True)])
def test_large_sets(bits, dtype, master):
    """sizes whose loads and stores go past the caches, clipped by a norm that is joined in a launch of its own"""
    from remixfusion_amd.optim import AdamW
    T = DTYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(19)
    sizes = [11_000_003, 257, 40]                                                  # >= 64 MB in each of these forms
    ps = [torch.nn.Parameter(torch.randn(n, device="cuda", generator=gen).mul(0.3).to(T)) for n in sizes]
    opt = AdamW(ps, **SETTINGS[1], state_bits=bits, master_weights=master, seed=5, max_grad_norm=3.0)
    refs = [Ref(p.detach().float().cpu().numpy(), bits, i, 5) for i, p in enumerate(ps)]
    for it in range(2):
        for p in ps:
            p.grad = magnitudes(p.numel(), gen).to(T)
        opt.step()
        grads = [p.grad.double() for p in ps]
        norm = math.sqrt(sum(float((g * g).sum()) for g in grads))
        assert abs(float(opt.grad_norm) - norm) <= (U + 1e-12) * norm and norm > 3.0
        for p, g, ref in zip(ps, grads, refs):
            tp, tm, tv = ref.step(g.cpu().numpy(), **SETTINGS[1], c=3.0 / (norm + 1e-6), half=U if master else half_eps(T))
            st = opt.state[p]
            if bits == 8:
                _check_code(st, ref, it)
            else:
                near(st["exp_avg"], ref.m, tm, "m"); near(st["exp_avg_sq"], ref.v, 2 * tv, "v")
                ref.m, ref.v = (st[k].double().cpu().numpy() for k in ("exp_avg", "exp_avg_sq"))
            near(st["master"] if master else p, ref.p, tp, "p")
            ref.p = (st["master"] if master else p.detach()).double().cpu().numpy()
    for p, ref, a, b in zip(ps, refs, *opt.moments()):
        near(a, ref.m, 0.0, "moments"); near(b, ref.v, U * np.abs(ref.v) + 2.0 ** -149, "moments")


def test_many_tensors_clipped():
    """more partial results than a wave joins by itself: the step and clip_grad_norm_ against the formula"""
    from remixfusion_amd.optim import AdamW, clip_grad_norm_
    gen = torch.Generator(device="cuda").manual_seed(29)
    ps = [torch.nn.Parameter(torch.randn(5000 + i, device="cuda", generator=gen)) for i in range(300)]
    for p in ps:
        p.grad = torch.randn(p.shape, device="cuda", generator=gen)
    old, before = [p.grad.clone() for p in ps], [p.detach().clone() for p in ps]
    norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in old))
    opt = AdamW(ps, lr=0.1, betas=(0.5, 0.9), eps=1.0, weight_decay=0.0, max_grad_norm=10.0)
    opt.step()
    assert abs(float(opt.grad_norm) - norm) <= (U + 1e-12) * norm
    c = 10.0 / (norm + 1e-6)
    for p, g, x in zip(ps, old, before):                       # first step: m / (1 - b1) = c g, sqrt(v / (1 - b2)) = |c g|
        want = x.double() - 0.1 * c * g.double() / (c * g.double().abs() + 1.0)
        assert float((p.detach().double() - want).abs().max()) <= 4 * U * 8
    for kind in (2.0, math.inf):
        for p, g in zip(ps, old):
            p.grad = g.clone()
        n = clip_grad_norm_(ps, 1.0, kind)
        want = norm if kind == 2.0 else max(float(g.abs().max()) for g in old)
        assert abs(float(n) - want) <= (U + 1e-12) * want
        for p, g in zip(ps, old):
            assert float((p.grad.double() - g.double() / (want + 1e-6)).abs().max()) <= 3 * U * 8


def test_numbers_of_other_types_in_the_groups():
    """what a configuration file or numpy makes of the settings: 8.0 is 8, and a scalar is a float"""
    from remixfusion_amd.optim import AdamW
    ps = [torch.nn.Parameter(torch.linspace(-1, 1, 777, device="cuda")) for _ in range(2)]
    a = AdamW([ps[0]], lr=np.float32(0.25), betas=(0.5, 0.75), eps=1e-8, weight_decay=0, state_bits=8.0, seed=3.0, master_weights=0, maximize=1)
    b = AdamW([ps[1]], lr=0.25, betas=(0.5, 0.75), weight_decay=0.0, state_bits=8, seed=3, maximize=True)
    for p, o in zip(ps, (a, b)):
        p.grad = torch.ones_like(p)
        o.step(); o.step()
    assert torch.equal(ps[0], ps[1]) and torch.equal(a.state[ps[0]]["exp_avg"], b.state[ps[1]]["exp_avg"])
    a.param_groups[0]["lr"] = None
    with pytest.raises(TypeError):
        a.step()
    a.param_groups[0]["lr"] = 0.25
    del a.param_groups[0]["eps"]
    with pytest.raises(KeyError):
        a.step()
    assert torch.equal(ps[0], ps[1]) and float(a.state[ps[0]]["step"]) == 2.0


def test_what_autograd_and_others_notice():
    """a step and a clipping raise the versions of what they write; a count that two parameters share is not raised twice"""
    from remixfusion_amd.optim import AdamW, clip_grad_norm_
    p, q = (torch.nn.Parameter(torch.ones(5, device="cuda")) for _ in range(2))
    opt = AdamW([p, q], lr=0.1, capturable=True)
    y = (p * p * q).sum()
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    v = p.grad._version
    clip_grad_norm_([p], 0.5)
    assert p.grad._version > v
    opt.step()
    with pytest.raises(RuntimeError):
        y.backward()                                           # its saved p is not what it was
    step = torch.tensor(3.0)
    for cap in (False, True):
        o = AdamW([p, q], lr=0.1, capturable=cap)
        st = {"exp_avg": torch.zeros(5, device="cuda"), "exp_avg_sq": torch.zeros(5, device="cuda")}
        o.load_state_dict({"state": {i: {"step": step, **{k: t.clone() for k, t in st.items()}} for i in range(2)},
                           "param_groups": o.state_dict()["param_groups"]})
        p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
        o.step(); o.step()
        assert [float(o.state[x]["step"]) for x in (p, q)] == [5.0, 5.0]


def test_against_torchs_adamw():
    """the fp32 step is torch.optim.AdamW's, and its state is read by torch and from torch"""
    from remixfusion_amd.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(8)
    a = [torch.nn.Parameter(torch.randn(s, device="cuda", generator=gen)) for s in ((32, 81), (6,), (1 << 16, 2), (4099,))]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    ours, ref = AdamW(a, **SETTINGS[1]), torch.optim.AdamW(b, **SETTINGS[1], foreach=False, fused=False)
    for it in range(5):
        for p, q in zip(a, b):
            p.grad = magnitudes(p.numel(), gen).reshape(p.shape)
            q.grad = p.grad.clone()
        ours.step(); ref.step()
        for p, q in zip(a, b):                     # each side is within 17 u of the step and 2 u of p of the exact one, every step
            tol = (it + 1) * (4 * U * q.detach().abs() + 40 * U * SETTINGS[1]["lr"] * 10)
            assert bool(((p - q).abs() <= tol).all()), it
    third = torch.optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in a], **SETTINGS[1])
    third.load_state_dict(ours.state_dict())
    assert torch.equal(third.state[third.param_groups[0]["params"][0]]["exp_avg"], ours.state[a[0]]["exp_avg"])
    fourth = AdamW(b, **SETTINGS[1])
    fourth.load_state_dict(ref.state_dict())
    for p, q in zip(a, b):
        p.grad = q.grad = torch.ones_like(p)
    fourth.step()
    assert float(fourth.state[b[0]]["step"]) == 6.0


@pytest.mark.parametrize("bits", [32, 8])
def test_values_that_are_not_finite(bits):
    """32 bits: only their own elements suffer; 8 bits: their run of 256 reads as NaN from the next step on, its neighbours do not"""
    from remixfusion_amd.optim import AdamW
    for bad in (math.inf, -math.inf, math.nan):
        p = torch.nn.Parameter(torch.ones(1000, device="cuda"))
        opt = AdamW([p], lr=0.1, state_bits=bits, weight_decay=0.0)
        p.grad = torch.full_like(p, 0.5)
        p.grad[300] = bad
        opt.step()
        fine = torch.ones(1000, dtype=torch.bool, device="cuda")
        fine[300] = False
        assert bool(torch.isfinite(p[fine]).all()) and not bool(torch.isfinite(p[300]))
        p.grad = torch.full_like(p, 0.5)
        opt.step()
        if bits == 8:
            fine[256:512] = False
            assert opt.state[p]["exponents"][:, 1].tolist() == [-128, -128] and bool((opt.state[p]["exponents"][:, [0, 2, 3]] != -128).all())
            assert bool(torch.isnan(opt.moments()[0][0][256:512]).all()) and bool(torch.isnan(p[256:512]).all())
        assert bool(torch.isfinite(p[fine]).all()) and not bool(torch.isfinite(p[300]))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("decay", [0.0, 0.1])
def test_parameters_that_are_not_finite(bits, dtype, decay):
    """inf (1 - lr wd) - update is inf, NaN stays NaN, and a half-precision parameter that a step carries over the edge is inf: as torch's"""
    from remixfusion_amd.optim import AdamW
    x = torch.full((600,), 1.0, device="cuda")
    x[3], x[300], x[301], x[599] = math.inf, -math.inf, math.nan, 65000.0
    p, q = (torch.nn.Parameter(x.to(DTYPES[dtype])) for _ in range(2))
    p.grad, q.grad = (torch.full_like(p, -0.5) for _ in range(2))
    lr = 2000.0 if dtype == "f16" else 0.01                     # 65000 + 2000 is no fp16
    a, b = AdamW([p], lr=lr, weight_decay=decay / lr, state_bits=bits), torch.optim.AdamW([q], lr=lr, weight_decay=decay / lr, foreach=False)
    for _ in range(2):
        a.step(); b.step()
        assert torch.equal(torch.isnan(p), torch.isnan(q)) and torch.equal(torch.isinf(p), torch.isinf(q))
        assert torch.equal(torch.sign(p.detach()).nan_to_num(9.0), torch.sign(q.detach()).nan_to_num(9.0))
    assert math.isinf(float(p.detach()[3])) and math.isinf(float(p.detach()[300])) and bool(torch.isinf(p[599])) == (dtype == "f16" and decay == 0.0)


def test_eight_bits_over_the_whole_range():
    """gradients from the smallest subnormal to the largest finite number, runs of zeros, runs of one value"""
    from remixfusion_amd.optim import AdamW
    rows = [np.zeros(256), np.full(256, 2.0 ** -149), np.full(256, 3e38), np.full(256, -1e-30), np.geomspace(1e-44, 1e18, 256),
            np.where(np.arange(256) == 7, 1e3, 0.0), np.where(np.arange(256) == 200, -1.0, 2.0 ** -17 * np.arange(256)),
            np.float32(1.875) * 2.0 ** (np.arange(256) // 8 - 16), np.nextafter(np.float32(1.875), np.float32(0)) * np.ones(256), -np.geomspace(1e-12, 1, 256)]
    g = np.concatenate(rows + [np.full(77, 1e-3)]).astype(np.float32)
    p = torch.nn.Parameter(torch.zeros(len(g), device="cuda"))
    opt = AdamW([p], lr=1e-3, betas=(0.9, 0.999), state_bits=8, weight_decay=0.0, seed=5)
    ref = Ref(np.zeros(len(g)), 8, 0, 5)
    for it in range(4):
        if it == 2:
            g = np.roll(g, 128) * np.float32(0.25)                    # runs mix: large next to small
        if it == 3:
            g = g * np.float32(0.0)                                   # nothing but decay
        p.grad = torch.from_numpy(g.copy()).cuda()
        opt.step()
        ref.step(g, 1e-3, (0.9, 0.999), 1e-8, 0.0)
        _check_code(opt.state[p], ref, it)
        live = ref.v > 0
        assert bool((opt.state[p]["exp_avg_sq"].cpu().numpy()[live] > 0).all())
        assert bool(torch.isfinite(p).all()) and float(p.detach().abs().max()) <= 1e-3 * (it + 1) * 40     # m without its v would be m / eps


@pytest.mark.parametrize("eps", [1e-15, 1e-8])
def test_eight_bit_states_of_any_bytes(eps):
    """every code under every exponent, moments that no run of steps leaves (m without v, roots beyond fp32's range): the step is the
    formula's.  m / eps may be of any size, so the tolerance is relative to the update."""
    from remixfusion_amd.optim import AdamW
    rng = np.random.default_rng(77)
    n = 256 * 600 + 131
    rows = -(-n // 256)
    cm, cv = rng.integers(0, 256, n, dtype=np.uint8), rng.integers(0, 256, n, dtype=np.uint8)
    cv[rng.random(n) < 0.2] = 0
    e1 = rng.integers(-127, 100, rows).astype(np.int8)
    e2 = np.clip(e1 + rng.integers(-3, 4, rows), -127, 127).astype(np.int8)
    g = np.where(rng.random(n) < 0.5, 0.0, rng.standard_normal(n) * np.repeat(2.0 ** np.clip(e1.astype(float), -120, 100), 256)[:n]).astype(np.float32)
    p = torch.nn.Parameter(torch.from_numpy(rng.standard_normal(n).astype(np.float32)).cuda())
    ref = Ref(p.detach().cpu().numpy(), 8, 0, 13)
    ref.k, ref.m, ref.v = 30, decode(cm, e1, 15), decode(cv, e2, 31)
    opt = AdamW([p], lr=1e-3, betas=(0.9, 0.99), eps=eps, weight_decay=0.01, state_bits=8, seed=13)
    state = {"step": torch.tensor(30.0), "exp_avg": torch.from_numpy(cm).cuda(), "exp_avg_sq": torch.from_numpy(cv).cuda(),
             "exponents": torch.from_numpy(np.stack([e1, e2])).cuda()}
    opt.load_state_dict({"state": {0: state}, "param_groups": opt.state_dict()["param_groups"]})
    p.grad = torch.from_numpy(g).cuda()
    old = ref.p.copy()
    opt.step()
    tp, _, _ = ref.step(g, 1e-3, (0.9, 0.99), eps, 0.01)
    _check_code(opt.state[p], ref, eps)
    # m is formed in fp64 here (4 u of each of its terms do not arise), rounded to fp32 once; what fp32 cannot hold is inf on the way out
    up = np.abs(ref.p - old * (1 - 1e-5))
    tol = U * (np.abs(old) + np.abs(ref.p)) + 16 * U * up + 2.0 ** -140
    fits = np.abs(ref.p) < 1e37
    got = p.detach().double().cpu().numpy()
    assert int((~fits).sum()) < n // 2
    bad = fits & ~(np.abs(got - ref.p) <= tol)
    assert not bad.any(), [(int(i), got[i], ref.p[i], tol[i]) for i in np.flatnonzero(bad)[:4]]


def test_rounding_is_unbiased_and_an_average_keeps_moving():
    """A code's expectation is the value itself: over 4096 seeds the mean is within 6 sigma of it, sigma <= step / 2 / sqrt(4096).
    And v of a constant gradient grows to g^2 although one step's change (1/1000) is far below the format's (1/8): with
    rounding to nearest it would stop where half a unit of the last place exceeds the increment."""
    from remixfusion_amd.optim import AdamW
    x = np.float32(0.0371)
    n = 4096
    ps = [torch.nn.Parameter(torch.zeros(256, device="cuda")) for _ in range(16)]
    sums, count = 0.0, 0
    for seed in range(n // 256):
        opt = AdamW(ps, state_bits=8, betas=(0.5, 0.5), seed=seed)
        for p in ps:
            p.grad = torch.full_like(p, float(x))
            p.grad[0] = 1.0                                            # the run's scale
        opt.step()
        avg, _ = opt.moments()
        sums += sum(float(a[1:].double().sum()) for a in avg)
        count += 255 * 16
    want = 0.5 * float(x)
    step = 2.0 ** (math.floor(math.log2(want)) - 3)
    assert abs(sums / count - want) <= 6 * step / 2 / math.sqrt(count), (sums / count, want)
    p = torch.nn.Parameter(torch.zeros(256 * 64, device="cuda"))
    opt = AdamW([p], lr=0.0, state_bits=8, betas=(0.9, 0.99), seed=3)
    p.grad = torch.full_like(p, 0.02)
    p.grad[::256] = 1.0
    for _ in range(600):
        opt.step()
    v = opt.moments()[1][0].double().reshape(-1, 256)[:, 1:].mean()
    want = 0.02 ** 2 * (1 - 0.99 ** 600)
    # the stationary spread of one element: each step adds a rounding of at most (v/8)^2/4, an average over ~1/(2 (1-b2)) of them:
    # sigma^2 <= (v/16)^2 * 50 -> sigma <= 0.45 v per element, 16320 elements: 6 sigma of the mean is 0.021 v
    assert abs(float(v) - want) <= 0.022 * want, (float(v), want)


def test_strides_gaps_and_ragged_gradients():
    """dense tensors in any order of dimensions, parameters with gaps in memory, gradients in another order than their parameter"""
    from remixfusion_amd.optim import AdamW
    for bits in (32, 8):
        gen = torch.Generator(device="cuda").manual_seed(2)
        base = torch.randn(40, 50, device="cuda", generator=gen)
        wide = torch.randn(40, 64, device="cuda", generator=gen)
        wide0 = wide.clone()
        last = torch.randn(2, 3, 5, 7, device="cuda", generator=gen).to(memory_format=torch.channels_last)
        ps = [torch.nn.Parameter(base.t().clone(memory_format=torch.preserve_format)), torch.nn.Parameter(wide[:, 3:53]), torch.nn.Parameter(last),
              torch.nn.Parameter(torch.randn(1, 33, device="cuda", generator=gen)), torch.nn.Parameter(torch.tensor(0.5, device="cuda"))]
        assert not ps[0].is_contiguous() and not ps[1].is_contiguous() and not ps[2].is_contiguous()
        qs = [torch.nn.Parameter(p.detach().clone(memory_format=torch.contiguous_format)) for p in ps]
        ours, ref = AdamW(ps, lr=1e-2, state_bits=bits), torch.optim.AdamW(qs, lr=1e-2)
        for it in range(2):
            for k, (p, q) in enumerate(zip(ps, qs)):
                g = torch.randn(p.shape, device="cuda", generator=gen) + 2.0
                q.grad = g
                p.grad = g if it else torch.empty_like(p).copy_(g)                # contiguous, or in the parameter's order
                if k == 3:
                    p.grad = torch.as_strided(g.clone(), (1, 33), (77, 1))           # a size-1 dimension's stride means nothing
            ours.step(); ref.step()
        # the same update up to fp32 (32 bits); 8-bit moments of gradients near 2 are off by a sixteenth at most, so a step by an eighth
        tol = 1e-6 if bits == 32 else 2 * 1e-2 * 0.2
        for p, q in zip(ps, qs):
            assert float((p - q).abs().max()) <= tol + 1e-6 * float(q.abs().max())
        assert torch.equal(wide[:, :3], wide0[:, :3]) and torch.equal(wide[:, 53:], wide0[:, 53:])


@pytest.mark.parametrize("shift", [0, 1, 4])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_nothing_around_the_tensors_is_touched(dtype, bits, shift):
    """parameters, gradients, moments, exponents and master copies inside larger buffers, at every kind of alignment: what lies before and
    behind stays as it was, and the step is the one of tensors of their own"""
    from remixfusion_amd.optim import AdamW
    T, n = DTYPES[dtype], 5000 + 3
    gen = torch.Generator(device="cuda").manual_seed(40)
    rows = -(-n // 256)

    def inside(t, at):
        buf = torch.full((t.numel() + 2 * 64,), 77, dtype=t.dtype, device="cuda")
        view = buf[at + 16:at + 16 + t.numel()].view(t.shape)
        view.copy_(t)
        return buf, view

    init, grad = (torch.randn(n, device="cuda", generator=gen).to(T) for _ in range(2))
    kind = torch.float32 if bits == 32 else torch.uint8
    state = {"exp_avg": torch.zeros(n, device="cuda", dtype=kind), "exp_avg_sq": torch.zeros(n, device="cuda", dtype=kind)}
    if bits == 8:
        state["exponents"] = torch.full((2, rows), -127, device="cuda", dtype=torch.int8)
    if dtype != "f32":
        state["master"] = init.float()
    around, out = [], []
    for wrap in (False, True):
        p, g, st = init.clone(), grad.clone(), {k: v.clone() for k, v in state.items()}
        if wrap:
            bufs = {}
            bufs["p"], p = inside(p, shift)
            bufs["g"], g = inside(g, shift)
            for k in list(st):
                bufs[k], st[k] = inside(st[k], 4 * shift if bits == 8 and k in ("exp_avg", "exp_avg_sq") else shift)
        p = torch.nn.Parameter(p)
        p.grad = g
        opt = AdamW([p], lr=0.01, state_bits=bits, master_weights=dtype != "f32", seed=3)
        opt.load_state_dict({"state": {0: {"step": torch.tensor(0.0), **st}}, "param_groups": opt.state_dict()["param_groups"]})
        for _ in range(3):
            opt.step()
        if wrap:
            for k, v in st.items():
                assert opt.state[p][k].data_ptr() == v.data_ptr(), k               # stepped where it lies
            for k, buf in bufs.items():
                at = (4 * shift if bits == 8 and k in ("exp_avg", "exp_avg_sq") else shift) + 16
                size = {"exponents": 2 * rows}.get(k, n)
                assert bool((buf[:at] == 77).all()) and bool((buf[at + size:] == 77).all()), k
        out.append([p.detach().clone()] + [opt.state[p][k].clone() for k in st])
    for a, b in zip(*out):
        assert torch.equal(a.reshape(-1), b.reshape(-1))


def test_states_at_odd_addresses():
    """8-bit moments that were loaded from an address no word starts at are brought to one; an expanded gradient is read as what it stands for"""
    from remixfusion_amd.optim import AdamW
    p, q = (torch.nn.Parameter(torch.ones(700, device="cuda")) for _ in range(2))
    buf = torch.zeros(1500, dtype=torch.uint8, device="cuda")
    a, b = (AdamW([x], lr=0.1, state_bits=8) for x in (p, q))
    a.load_state_dict({"state": {0: {"step": torch.tensor(0.0), "exp_avg": buf[1:701], "exp_avg_sq": buf[703:1403],
                                     "exponents": torch.full((2, 3), -127, dtype=torch.int8, device="cuda")}},
                       "param_groups": a.state_dict()["param_groups"]})
    p.grad = torch.full((1,), 0.25, device="cuda").expand(700)
    q.grad = torch.full((700,), 0.25, device="cuda")
    a.step(); b.step()
    assert torch.equal(p, q) and torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"]) and int(buf.max()) == 0
    from remixfusion_amd import _lib as L
    from remixfusion_amd.optim import clip_grad_norm_
    with pytest.raises(L.RfxError):
        clip_grad_norm_([p], 1.0)                                                  # which cannot be written


def test_learning_rates_on_the_device():
    from remixfusion_amd.optim import AdamW
    p = torch.nn.Parameter(torch.ones(5, device="cuda"))
    p.grad = torch.ones_like(p)
    for lr in (torch.tensor(0.1), torch.tensor([0.1, 0.1], device="cuda"), torch.tensor(0.1, device="cuda", dtype=torch.float64)):
        with pytest.raises(ValueError):
            AdamW([p], lr=lr, capturable=True).step()
    assert float(p.detach().min()) == 1.0
    AdamW([p], lr=torch.tensor([0.1], device="cuda"), capturable=True, weight_decay=0.0).step()
    assert abs(float(p.detach()[0]) - 0.9) < 1e-6
    # eps below fp32's normal numbers, no gradient: nothing happens
    z = torch.nn.Parameter(torch.ones(300, device="cuda"))
    z.grad = torch.zeros_like(z)
    AdamW([z], state_bits=8, eps=1e-42, weight_decay=0.0).step()
    assert bool((z == 1).all())


def test_parameters_that_share_memory_step_one_after_the_other():
    from remixfusion_amd.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(4)
    a = torch.randn(9000, device="cuda", generator=gen)
    b = a.clone()
    ps, qs = ([torch.nn.Parameter(x[:6000]), torch.nn.Parameter(x[3500:]), torch.nn.Parameter(x[100:300])] for x in (a, b))
    for p, q in zip(ps, qs):
        p.grad = q.grad = torch.randn(p.shape, device="cuda", generator=gen)
    ours, ref = AdamW(ps, lr=0.1), torch.optim.AdamW(qs, lr=0.1, foreach=False)
    ours.step(); ref.step()
    assert float((a - b).abs().max()) <= 2e-6                                    # three steps of 0.1 and roundings of values near 4


def test_refusals_on_the_device():
    from remixfusion_amd import _lib as L
    from remixfusion_amd.optim import AdamW, clip_grad_norm_
    p = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    q = torch.nn.Parameter(torch.zeros(8))
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    with pytest.raises(L.RfxError):
        AdamW([p, q]).step()
    with pytest.raises(L.RfxError):
        AdamW([q, p]).step()
    d = torch.nn.Parameter(torch.zeros(8, device="cuda", dtype=torch.float64))
    d.grad = torch.ones_like(d)
    with pytest.raises(L.RfxError):
        AdamW([d]).step()
    with pytest.raises(L.RfxError):
        clip_grad_norm_([d], 1.0)
    with pytest.raises(L.RfxError):
        clip_grad_norm_([p], 1.0, norm_type=1.0)
    with pytest.raises(L.RfxError):
        clip_grad_norm_([p, q], 1.0)
    e = torch.nn.Parameter(torch.zeros(1, device="cuda").expand(8))
    e.grad = torch.ones(8, device="cuda")
    with pytest.raises(L.RfxError):
        AdamW([e]).step()
    s = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    s.grad = torch.ones(8, device="cuda").to_sparse()
    with pytest.raises(L.RfxError):
        AdamW([s]).step()
    opt = AdamW([p], state_bits=8)
    opt.step()
    sd = copy.deepcopy(opt.state_dict())
    for key, value in (("exp_avg", torch.zeros(8, device="cuda")), ("exponents", torch.zeros(2, 2, dtype=torch.int8, device="cuda")),
                       ("exp_avg_sq", torch.zeros(9, dtype=torch.uint8, device="cuda"))):
        bad = copy.deepcopy(sd)
        bad["state"][0][key] = value
        with pytest.raises(L.RfxError):
            AdamW([p], state_bits=8).load_state_dict(bad)
    bad = copy.deepcopy(sd)
    bad["param_groups"][0]["state_bits"] = 32
    with pytest.raises(L.RfxError):
        AdamW([p]).load_state_dict(bad)
    before = p.detach().clone()
    g = torch.cuda.CUDAGraph()
    plain = AdamW([p])
    plain.step()
    before = p.detach().clone()
    with pytest.raises(L.RfxError):
        with torch.cuda.graph(g):
            plain.step()
    torch.cuda.synchronize()
    assert torch.equal(p.detach(), before)


def test_states_that_change_between_steps_are_noticed():
    """gradients that come and go, parameters and states that are replaced, groups that join, counts that differ"""
    from remixfusion_amd.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(6)

    def both(n):
        x = torch.randn(n, device="cuda", generator=gen)
        return torch.nn.Parameter(x.clone()), torch.nn.Parameter(x.clone())

    (a, x), (b, y), (c, z) = both(300), both(5000), both(77)
    ours, ref = AdamW([a, b], lr=0.01), torch.optim.AdamW([x, y], lr=0.01, foreach=False)

    def step(pairs):
        for p, q in ((a, x), (b, y), (c, z)):
            p.grad = q.grad = None
        for p, q in pairs:
            p.grad = torch.randn(p.shape, device="cuda", generator=gen)
            q.grad = p.grad.clone()
        ours.step(); ref.step()
        for p, q in ((a, x), (b, y), (c, z)):
            assert float((p - q).abs().max()) <= 3e-6

    step([(a, x)])
    step([(a, x), (b, y)])                                   # b's first step is a's second
    assert float(ours.state[a]["step"]) == 2.0 and float(ours.state[b]["step"]) == 1.0
    step([(b, y)])
    step([])
    ours.add_param_group({"params": [c], "lr": 0.05}); ref.add_param_group({"params": [z], "lr": 0.05})
    step([(a, x), (b, y), (c, z)])
    assert [float(ours.state[p]["step"]) for p in (a, b, c)] == [3.0, 3.0, 1.0]
    a.data, x.data = a.data.clone() * 2, x.data.clone() * 2
    step([(a, x), (c, z)])
    for o, ps in ((ours, (a, b, c)), (ref, (x, y, z))):
        for p in ps:
            for k in ("exp_avg", "exp_avg_sq"):
                o.state[p][k] = o.state[p][k].clone() * 0.5
    step([(a, x), (b, y), (c, z)])
    for o, p in ((ours, b), (ref, y)):
        o.state[p]["exp_avg"].data = o.state[p]["exp_avg"].data.clone() * 0.25
    step([(a, x), (b, y), (c, z)])
    ours.state.clear(); ref.state.clear()
    step([(a, x), (b, y)])
    assert float(ours.state[a]["step"]) == 1.0
    b.data, y.data = b.data[:100].clone(), y.data[:100].clone()       # another size: the old state does not fit and is not used
    from remixfusion_amd import _lib as L
    b.grad = torch.ones_like(b)
    with pytest.raises(L.RfxError):
        ours.step()


def test_eight_bit_state_survives_a_checkpoint(tmp_path):
    from remixfusion_amd.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(1)
    init = [torch.randn(n, device="cuda", generator=gen).bfloat16() for n in (3, 700, 5001)]
    grads = [[torch.randn(t.shape, device="cuda", generator=gen).bfloat16() for t in init] for _ in range(6)]

    def run(upto, ps, opt, first=0):
        for k in range(first, upto):
            for p, g in zip(ps, grads[k]):
                p.grad = g
            opt.step()

    make = lambda: [torch.nn.Parameter(t.clone()) for t in init]                     # noqa: E731
    kw = dict(lr=0.01, state_bits=8, master_weights=True, seed=21)
    ps = make()
    whole = AdamW(ps, **kw)
    run(6, ps, whole)
    qs = make()
    opt = AdamW(qs, **kw)
    run(3, qs, opt)
    torch.save({"opt": opt.state_dict(), "p": [q.detach() for q in qs]}, tmp_path / "ck.pt")
    ck = torch.load(tmp_path / "ck.pt", weights_only=True)
    rs = [torch.nn.Parameter(t.cuda()) for t in ck["p"]]
    back = AdamW(rs, lr=0.5)                                                         # the saved groups say what they are
    back.load_state_dict(ck["opt"])
    assert back.param_groups[0]["state_bits"] == 8 and back.state[rs[1]]["master"].dtype == torch.float32
    run(6, rs, back, 3)
    twin = copy.deepcopy(opt)
    ts = twin.param_groups[0]["params"]
    run(6, ts, twin, 3)
    for p, r, t in zip(ps, rs, ts):
        assert torch.equal(p, r) and torch.equal(p, t)
        for key in ("exp_avg", "exp_avg_sq", "exponents", "master"):
            assert torch.equal(whole.state[p][key], back.state[r][key]) and torch.equal(whole.state[p][key], twin.state[t][key])


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_clip_grad_norm(norm_type):
    """against fp64: N is summed in fp64 and rounded once; a gradient gets one fp32 product and one rounding to its type"""
    from remixfusion_amd.optim import clip_grad_norm_
    gen = torch.Generator(device="cuda").manual_seed(12)
    sizes = [1, 2, 3, 5, 0, 1000, 4097, 16384, 16385, 40001, 300000] + [17] * 140             # more tensors than a launch takes
    types = [torch.float32, torch.bfloat16, torch.float16]
    buf = [magnitudes(n + 1, gen).to(types[i % 3]) for i, n in enumerate(sizes)]
    for limit in (1e-3, 1e9):
        ps = []
        for i, b in enumerate(buf):
            g = b.clone()[1:] if i % 2 else b[:-1].clone()                                    # every other one off any vector's alignment
            ps.append(torch.nn.Parameter(torch.zeros_like(g)))
            ps[-1].grad = g
        old = [p.grad.double().cpu().numpy() for p in ps]
        want = max(np.abs(o).max(initial=0.0) for o in old) if norm_type == math.inf else math.sqrt(sum((o * o).sum() for o in old))
        norm = clip_grad_norm_(ps, limit, norm_type)
        assert norm.dtype == torch.float32 and abs(float(norm) - want) <= (U + 1e-12) * want
        c = min(1.0, limit / (want + 1e-6))
        for p, o in zip(ps, old):
            tiny = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}[p.dtype]
            tol = (half_eps(p.dtype) + 3 * U) * np.abs(o * c) + tiny if c < 1 else 0.0
            near(p.grad, o * c, tol, (limit, p.dtype, p.numel()))
        for p, o in zip(ps, old):
            p.grad = torch.from_numpy(o).to(p.dtype).cuda()
        again = clip_grad_norm_(ps, limit, norm_type)
        assert torch.equal(again, norm)                                                      # the order of the sum is fixed


def test_clip_of_odd_sets():
    from remixfusion_amd.optim import clip_grad_norm_
    p = torch.nn.Parameter(torch.zeros(4, 6, device="cuda"))
    p.grad = torch.arange(24.0, device="cuda").reshape(6, 4).t()                              # another order of dimensions
    q = torch.nn.Parameter(torch.zeros(4, 3, device="cuda"))
    wide = torch.ones(4, 8, device="cuda")
    q.grad = wide[:, 2:5]                                                                      # gaps
    old = p.grad.clone()
    n = clip_grad_norm_([p, q], 1.0)
    want = math.sqrt(float((old.double() ** 2).sum()) + 12)
    assert abs(float(n) - want) < 1e-5 and float((p.grad - old / want).abs().max()) < 1e-5
    assert float((q.grad - 1 / want).abs().max()) < 1e-7 and float(wide[:, :2].min()) == 1.0 and float(wide[:, 5:].min()) == 1.0
    r = torch.nn.Parameter(torch.zeros(100000, device="cuda"))
    r.grad = torch.ones(100000, device="cuda")
    s = torch.nn.Parameter(torch.zeros(100000, device="cuda"))
    s.grad = torch.ones(100000, device="cuda")
    a, b = clip_grad_norm_([r, r], 1.0), torch.nn.utils.clip_grad_norm_([s, s], 1.0, foreach=False)      # twice in the list: twice in the norm, scaled twice
    assert abs(float(a) - float(b)) < 1e-3 and float((r.grad / s.grad - 1).abs().max()) < 1e-5
    for bad, factor in ((math.inf, 0.0), (math.nan, math.nan)):
        t = torch.nn.Parameter(torch.zeros(300, device="cuda"))
        for kind in (2.0, math.inf):
            t.grad = torch.ones(300, device="cuda")
            t.grad[211] = bad
            before = t.grad.clone()
            with pytest.raises(RuntimeError):
                clip_grad_norm_(t, 1.0, kind, error_if_nonfinite=True)
            assert torch.equal(t.grad.nan_to_num(7.0), before.nan_to_num(7.0))
            n = clip_grad_norm_(t, 1.0, kind)
            assert not math.isfinite(float(n)) and math.isnan(float(t.grad[211]))
            near(t.grad[:211], np.full(211, factor), 0.0, "others")
    t.grad = torch.full((300,), 3e38, device="cuda")                                           # squares that no fp32 holds
    assert abs(float(clip_grad_norm_(t, 1.0)) / (3e38 * math.sqrt(300)) - 1) < 1e-6 or math.isinf(float(torch.tensor(3e38 * math.sqrt(300))))
    assert abs(float(t.grad[0]) * math.sqrt(300) - 1) < 1e-5
    t.grad = torch.full((300,), 1.0, device="cuda")
    clip_grad_norm_(t, 0.0)
    assert float(t.grad.abs().max()) == 0.0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_clipped_step_is_the_step_of_clipped_gradients(bits, dtype):
    """max_grad_norm against the oracle, gradients left alone, and grad_norm is clip_grad_norm_'s"""
    from remixfusion_amd.optim import AdamW, clip_grad_norm_
    T = DTYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(31)
    ps = [torch.nn.Parameter((torch.randn(n, device="cuda", generator=gen) * 0.3).to(T)) for n in (7, 300, 5000, 40003)]
    opt = AdamW(ps, **SETTINGS[0], state_bits=bits, max_grad_norm=0.25, seed=2)
    refs = [Ref(p.detach().float().cpu().numpy(), bits, i, 2) for i, p in enumerate(ps)]
    for it in range(3):
        for p in ps:
            p.grad = (magnitudes(p.numel(), gen) * (10.0 if it < 2 else 1e-6)).to(T)
        old = [p.grad.clone() for p in ps]
        opt.step()
        norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in old))
        c = min(1.0, 0.25 / (norm + 1e-6))
        assert (c < 1) == (it < 2) and abs(float(opt.grad_norm) - norm) <= (U + 1e-12) * norm
        for p, ref, g in zip(ps, refs, old):
            assert torch.equal(p.grad, g)
            tp, tm, tv = ref.step(g.float().cpu().numpy(), **SETTINGS[0], c=c, half=half_eps(T))
            st = opt.state[p]
            if bits == 8:
                _check_code(st, ref, it)
            else:
                near(st["exp_avg"], ref.m, tm, "m"); near(st["exp_avg_sq"], ref.v, 2 * tv, "v")
                ref.m, ref.v = (st[k].double().cpu().numpy() for k in ("exp_avg", "exp_avg_sq"))
            near(p, ref.p, tp, "p")
            ref.p = p.detach().double().cpu().numpy()
    n = clip_grad_norm_(ps, 0.25)
    assert torch.equal(n, opt.grad_norm)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_replay_like_eager_ones(bits):
    """capturable: the count and the learning rate live on the device; replays with other work between them, two graphs at once"""
    from remixfusion_amd.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(17)
    init = [torch.randn(n, device="cuda", generator=gen) for n in (5, 700, 9001)] + [torch.randn(333, device="cuda", generator=gen).bfloat16()]

    def make(lr):
        ps = [torch.nn.Parameter(t.clone()) for t in init]
        for p in ps:
            p.grad = torch.zeros_like(p)
        return ps, AdamW([dict(params=ps[:2]), dict(params=ps[2:], weight_decay=0.2)], lr=lr, state_bits=bits, capturable=True, master_weights=True,
                         max_grad_norm=0.5, seed=8)

    lr = torch.tensor(0.01, device="cuda")
    (ps, opt), (qs, ref), (rs, other) = make(lr), make(lr), make(lr)
    opt.prepare(), other.prepare()
    graphs = []
    for o in (opt, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o.step()
        graphs.append((g, o.grad_norm))
    for p in ps + rs:
        assert float(p.detach().float().abs().max()) > 0
    for it in range(6):
        lr.fill_(0.01 / (it + 1))
        for k, (p, q, r) in enumerate(zip(ps, qs, rs)):
            x = torch.randn(p.shape, device="cuda", generator=gen).to(p.dtype)
            p.grad.copy_(x); q.grad.copy_(x); r.grad.copy_(x)
        graphs[0][0].replay()
        if it % 2:
            torch.cuda.synchronize()
            torch.randn(1 << 20, device="cuda").sum().item()              # eager work in between
        graphs[1][0].replay()
        ref.step()
        for p, q, r in zip(ps, qs, rs):
            assert torch.equal(p, q) and torch.equal(r, q), it
            for key, t in ref.state[q].items():
                assert torch.equal(opt.state[p][key], t) and torch.equal(other.state[r][key], t), (it, key)
        assert torch.equal(graphs[0][1], ref.grad_norm) and torch.equal(graphs[1][1], ref.grad_norm)
        assert float(opt.state[ps[0]]["step"]) == it + 1
    plain = [torch.nn.Parameter(t.clone()) for t in init]                  # the host's count gives the same steps
    for p in plain:
        p.grad = torch.randn(p.shape, device="cuda", generator=gen).to(p.dtype)
    fresh = [torch.nn.Parameter(t.clone()) for t in init]
    for p, q in zip(fresh, plain):
        p.grad = q.grad
    a, b = AdamW(plain, lr=0.01, state_bits=bits), AdamW(fresh, lr=0.01, state_bits=bits, capturable=True)
    for _ in range(3):
        a.step(); b.step()
    for p, q in zip(plain, fresh):
        assert float((p - q).detach().abs().max()) <= 4 * half_eps(p.dtype) * 4
        assert torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"])


def test_clipping_and_reading_back_in_a_graph():
    """clip_grad_norm_, step and moments() as one captured run, replayed on new gradients, against the same calls outside"""
    from remixfusion_amd.optim import AdamW, clip_grad_norm_
    gen = torch.Generator(device="cuda").manual_seed(37)
    sizes = [3, 1000, 20001]
    init = [torch.randn(n, device="cuda", generator=gen) for n in sizes]

    def make():
        ps = [torch.nn.Parameter(t.clone()) for t in init]
        for p in ps:
            p.grad = torch.zeros_like(p)
        opt = AdamW(ps, lr=0.01, state_bits=8, capturable=True, seed=1)
        opt.prepare()
        return ps, opt

    def run(ps, opt):
        norm = clip_grad_norm_(ps, 0.5), clip_grad_norm_(ps, 1e9, math.inf)
        opt.step()
        return norm + tuple(opt.moments())

    (ps, opt), (qs, ref) = make(), make()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = run(ps, opt)
    for it in range(5):
        for p, q in zip(ps, qs):
            x = torch.randn(p.shape, device="cuda", generator=gen) * 10.0 ** (it - 3)         # over the limit, and under it
            p.grad.copy_(x); q.grad.copy_(x)
        g.replay()
        torch.ones(1 << 20, device="cuda").sum().item()
        out = run(qs, ref)
        assert torch.equal(held[0], out[0]) and torch.equal(held[1], out[1]), it
        for p, q, a, b, c, d in zip(ps, qs, held[2], out[2], held[3], out[3]):
            assert torch.equal(p, q) and torch.equal(p.grad, q.grad) and torch.equal(a, b) and torch.equal(c, d), it


def test_capture_needs_the_state_beforehand():
    from remixfusion_amd import _lib as L
    from remixfusion_amd.optim import AdamW
    p = torch.nn.Parameter(torch.ones(5, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = AdamW([p], capturable=True)
    with pytest.raises(L.RfxError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    torch.cuda.synchronize()
    opt.step()
    assert float(opt.state[p]["step"]) == 1.0 and opt.state[p]["step"].is_cuda


def test_work_on_another_stream():
    from remixfusion_amd.optim import AdamW
    gen = torch.Generator(device="cuda").manual_seed(23)
    init = torch.randn(500000, device="cuda", generator=gen)
    g = torch.randn(500000, device="cuda", generator=gen)
    out = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        p = torch.nn.Parameter(init.clone())
        opt = AdamW([p], lr=0.1, state_bits=8, max_grad_norm=1.0)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(5):
                p.grad = g.clone()
                opt.step()
            avg, _ = opt.moments()
        torch.cuda.current_stream().wait_stream(stream)
        out.append((p.detach().clone(), avg[0].clone(), opt.grad_norm.clone()))
    for x, y in zip(*out):
        assert torch.equal(x, y)


def test_elements_past_32_bits():
    """one tensor of 2^32 + 1003 elements: the last runs have to be the ones that a step of their own gives"""
    from remixfusion_amd.optim import AdamW, clip_grad_norm_
    n, tail = (1 << 32) + 1003, 1003 + 256 * 4
    p = torch.nn.Parameter(torch.full((n,), 0.5, device="cuda", dtype=torch.bfloat16))
    p.grad = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    gen = torch.Generator(device="cuda").manual_seed(3)
    p.grad[-tail:] = torch.randn(tail, device="cuda", generator=gen).bfloat16()
    p.grad[0] = 2.0
    opt = AdamW([p], lr=0.01, state_bits=8, seed=6, weight_decay=0.0)
    opt.step()
    g = p.grad[-tail:].float().cpu().numpy()
    ref = Ref(np.full(tail, 0.5), 8, 0, 6)
    tp, _, _ = ref.step(g, 0.01, (0.9, 0.999), 1e-8, 0.0, half=half_eps(torch.bfloat16), first=n - tail)
    near(p[-tail:], ref.p, tp, "p")
    st = opt.state[p]
    assert np.array_equal(st["exp_avg_sq"][-tail:].cpu().numpy(), ref.cv)
    assert np.array_equal(st["exponents"][:, -(-tail // 256):].cpu().numpy()[:, -len(ref.e1):], np.stack([ref.e1, ref.e2]))
    assert float(p[0]) < 0.5 and float(p[1]) == 0.5 and float(p[n // 2]) == 0.5 and int(st["exp_avg_sq"][1 << 20]) == 0
    norm = clip_grad_norm_([p], 1.0)
    want = math.sqrt(4.0 + float((g.astype(np.float64) ** 2).sum()))
    assert abs(float(norm) - want) <= 1e-6 * want and abs(float(p.grad[0]) - 2.0 / want) < 1e-2
    near(p.grad[-tail:], g / want, (2.0 ** -8 + 1e-6) * np.abs(g / want), "scaled")


def test_closure_and_zero_sized():
    from remixfusion_amd.optim import AdamW, clip_grad_norm_
    p, e = torch.nn.Parameter(torch.ones(5, device="cuda")), torch.nn.Parameter(torch.ones(0, 3, device="cuda"))
    opt = AdamW([e, p], lr=0.1, state_bits=8)

    def closure():
        opt.zero_grad()
        loss = (p * p).sum() + e.sum()
        loss.backward()
        return loss

    assert float(opt.step(closure).detach()) == 5.0 and float(p.detach().max()) < 1.0
    assert float(opt.state[e]["step"]) == 1.0
    assert abs(float(clip_grad_norm_([e, p], 10.0)) - math.sqrt(20)) < 1e-5
    only = AdamW([e])
    only.step()
    assert float(clip_grad_norm_([e], 1.0)) == 0.0 and [t.shape for t in only.moments()[0]] == [(0, 3)]


def test_adam_with_decoupled_decay_is_not_stepped_as_l2():
    """optim.Adam's native step folds the decay into the gradient: the decoupled kind takes torch's step"""
    from remixfusion_amd.optim import Adam
    p, q = (torch.nn.Parameter(torch.linspace(-1, 1, 100, device="cuda")) for _ in range(2))
    ours = Adam([p], lr=0.1, weight_decay=0.5, decoupled_weight_decay=True)
    ref = torch.optim.Adam([q], lr=0.1, weight_decay=0.5, decoupled_weight_decay=True)
    for _ in range(2):
        p.grad = q.grad = torch.full((100,), 0.25, device="cuda")
        ours.step(); ref.step()
    assert float((p - q).detach().abs().max()) <= 1e-6


@pytest.mark.parametrize("dtype", list(DTYPES.values()), ids=list(DTYPES))
@pytest.mark.parametrize("n", [3, 4099, 70001, 3000003])
def test_the_norm_does_not_depend_on_addresses(dtype, n):
    """all 64 bits of the norm: the order of its sum is one of sizes, not of where the gradients start"""
    from remixfusion_amd import _lib
    lib = _lib.load()
    g = (torch.randn(n, generator=torch.Generator().manual_seed(n)) * 0.3).to(dtype).cuda()
    ws = torch.empty(lib.rfx_grad_norm_workspace_bytes(1) // 8, dtype=torch.float64, device="cuda")
    seen = []
    for first in (0, 1, 2, 3, 5):
        at = torch.zeros(n + 8, dtype=dtype, device="cuda")[first:first + n].copy_(g)
        clip = torch.empty(2, dtype=torch.float64, device="cuda")
        row = (_lib.GradTensor * 1)(_lib.GradTensor(at.data_ptr(), n, _lib.DTYPES[dtype], 0))
        _lib.check(lib.rfx_grad_norm(row, 1, 2, 1.0, clip.data_ptr(), None, ws.data_ptr(), ws.numel() * 8, _lib.stream_ptr(0)), "rfx_grad_norm")
        seen.append(float(clip[0]))
    assert len(set(seen)) == 1, seen
    want = math.sqrt(float((g.cpu().double() ** 2).sum()))
    assert abs(seen[0] - want) <= 1e-12 * want


def test_the_norm_is_that_of_the_last_step():
    from remixfusion_amd.optim import AdamW
    p = torch.nn.Parameter(torch.ones(9, device="cuda"))
    opt = AdamW([p], max_grad_norm=1.0)
    for limit, grad, want in ((1.0, 2.0, 6.0), (None, 2.0, None), (5.0, 1.0, 3.0), (5.0, None, None), (0.0, 1.0, 3.0)):
        opt.max_grad_norm = limit
        p.grad = None if grad is None else torch.full_like(p, grad)
        opt.step()
        assert opt.grad_norm is None if want is None else float(opt.grad_norm) == want


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_that_parameters_share_is_parted(bits):
    """one set of moments (and master weights) given to two parameters, and one tensor as both moments: as if each had its own"""
    from remixfusion_amd.optim import AdamW
    n = 1000
    gen = torch.Generator(device="cuda").manual_seed(4)
    kind = torch.uint8 if bits == 8 else torch.float32
    m = torch.full((n,), 40, dtype=kind, device="cuda")
    st = {"step": torch.tensor(2.0), "exp_avg": m, "exp_avg_sq": m, "master": torch.randn(n, device="cuda", generator=gen)}
    if bits == 8:
        st["exponents"] = torch.zeros(2, 4, dtype=torch.int8, device="cuda")
    grads = [torch.randn(n, device="cuda", generator=gen).bfloat16() for _ in range(2)]
    out = []
    for share in (True, False):
        ps = [torch.nn.Parameter(torch.zeros(n, device="cuda", dtype=torch.bfloat16)) for _ in range(2)]
        opt = AdamW(ps, lr=0.1, state_bits=bits, master_weights=True)
        own = {k: t.clone() for k, t in st.items()}
        if share:
            own["exp_avg_sq"] = own["exp_avg"]
        opt.load_state_dict({"state": {i: dict(own) if share else {k: t.clone() for k, t in st.items()} for i in range(2)},
                             "param_groups": opt.state_dict()["param_groups"]})
        for _ in range(3):
            for p, g in zip(ps, grads):
                p.grad = g.clone()
            opt.step()
        out.append([t.clone() for p in ps for t in (p.detach(), *opt.state[p].values())])
    for a, b in zip(*out):
        assert torch.equal(a, b)


@pytest.mark.parametrize("what", ["order", "type", "count", "shared", "master"])
def test_a_capture_does_not_bring_a_state_over(what):
    """what an eager step would convert once, a graph would convert on every replay: refused, and nothing of the state is changed"""
    from remixfusion_amd import _lib as L
    from remixfusion_amd.optim import AdamW
    p, q = (torch.nn.Parameter(torch.ones(6, 4, device="cuda", dtype=torch.bfloat16)) for _ in range(2))
    opt = AdamW([p, q], capturable=True, master_weights=what == "master")
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    opt.step()
    st = opt.state[q]
    if what == "order":
        st["exp_avg"] = torch.zeros(4, 6, device="cuda").t()
    elif what == "type":
        st["exp_avg_sq"] = st["exp_avg_sq"].double()
    elif what == "count":
        st["step"] = torch.tensor(1.0)
    elif what == "shared":
        st["exp_avg"] = opt.state[p]["exp_avg"]
    else:
        del st["master"]
    torch.cuda.synchronize()
    before = {x: {k: (t, t.clone()) for k, t in opt.state[x].items()} for x in (p, q)}
    torch.cuda.synchronize()
    with pytest.raises(L.RfxError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    torch.cuda.synchronize()
    for x in (p, q):
        assert set(opt.state[x]) == set(before[x])
        for k, (t, value) in before[x].items():
            assert opt.state[x][k] is t and torch.equal(t, value)
    opt.step()                                                     # an eager one brings it over
    torch.cuda.synchronize()
    assert opt.state[q]["exp_avg"] is not opt.state[p]["exp_avg"]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert float(opt.state[q]["step"]) == 3.0


def test_a_state_may_hold_what_is_not_a_tensor():
    from remixfusion_amd.optim import AdamW
    p = torch.nn.Parameter(torch.ones(5, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = AdamW([p])
    opt.step()
    opt.state[p]["name"] = "decoder"
    opt.step(); opt.step()
    assert opt.state[p]["name"] == "decoder" and float(opt.state[p]["step"]) == 3.0
