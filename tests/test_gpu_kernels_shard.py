"""AdamW over many tensors and the sum of squares against references in 64 bits; the 8-bit states bit for bit."""
import math

import numpy as np
import pytest

import local_ref as ref

pytestmark = pytest.mark.gpu

SIZES = [1, 2, 3, 4, 5, 31, 32, 33, 63, 64, 65, 255, 256, 257, 1023, 1024, 1025, 2047, 2049, 4097, 70001]
HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, step=7)
GUARD = 64          # elements around every buffer that nothing may touch


def _types():
    import torch
    import rccl_amd as ra
    return {"f32": (ra.ncclFloat32, torch.float32), "bf16": (ra.ncclBfloat16, torch.bfloat16), "f16": (ra.ncclFloat16, torch.float16)}


def _np(t):
    import torch
    return t.to(torch.float64).cpu().numpy() if t.dtype != torch.uint8 else t.cpu().numpy()


class Case:
    """Tensors of `sizes` cut from flat buffers, each `shift` elements past a multiple of 32, with guards around them."""

    def __init__(self, sizes, param="f32", grad="f32", copy=None, mx=False, shift=0, seed=0, scale=1e-2):
        import torch
        self.torch, self.sizes, self.names, self.mx = torch, sizes, (param, grad, copy), mx
        ty, rng = _types(), np.random.default_rng(seed)
        starts, at = [], GUARD
        for n in sizes:
            starts.append(at + shift)
            at += -(-(n + shift + GUARD) // 32) * 32
        self.starts, total = starts, at + GUARD
        self.sstarts = [s // 32 for s in starts]
        flat = lambda x, t: torch.from_numpy(x.astype(np.float32)).to(t).cuda()  # noqa: E731
        self.loud = np.exp(rng.standard_normal(total))
        self.param = flat(rng.standard_normal(total), ty[param][1])
        self.grad = flat(scale * self.loud * rng.standard_normal(total), ty[grad][1])
        self.copy = flat(rng.standard_normal(total), ty[copy][1]) if copy else None
        m, v = 0.3 * scale * self.loud * rng.standard_normal(total), (scale * self.loud * (0.05 + np.abs(rng.standard_normal(total)))) ** 2
        if mx:
            self.m, self.v = (torch.from_numpy(rng.integers(0, 127, total, dtype=np.uint8)).cuda() for _ in range(2))
            self.m |= torch.from_numpy(rng.integers(0, 2, total, dtype=np.uint8) << 7).cuda()
            self.ms = torch.from_numpy(rng.integers(108, 112, total // 32 + 8, dtype=np.uint8)).cuda()
            self.vs = torch.from_numpy(rng.integers(108, 112, total // 32 + 8, dtype=np.uint8)).cuda()
        else:
            self.m, self.v, self.ms, self.vs = flat(m, torch.float32), flat(v, torch.float32), None, None
        self.bufs = [b for b in (self.param, self.grad, self.copy, self.m, self.v, self.ms, self.vs) if b is not None]

    def cut(self, buf, i):
        return buf[self.starts[i]:self.starts[i] + self.sizes[i]]

    def cut_scale(self, buf, i):
        return buf[self.sstarts[i]:self.sstarts[i] - (-self.sizes[i] // 32)]

    def table(self):
        import rccl_amd as ra
        rows = []
        for i in range(len(self.sizes)):
            rows.append(ra.adamw_tensor(self.cut(self.param, i), self.cut(self.grad, i), self.cut(self.m, i), self.cut(self.v, i),
                                        exp_avg_scale=self.cut_scale(self.ms, i) if self.mx else None, exp_avg_sq_scale=self.cut_scale(self.vs, i) if self.mx else None,
                                        copy=self.cut(self.copy, i) if self.copy is not None else None))
        return np.array(rows, dtype=np.int64).reshape(-1, 8)

    def snapshot(self):
        return [b.clone() for b in self.bufs]

    def run(self, **kw):
        import rccl_amd as ra
        p, g, c = self.names
        ty = _types()
        args = dict(HYPER, **kw)
        ra.adamw(self.table(), ty[p][0], ty[g][0], ty[c][0] if c else -1, ra.rcclAmdStateMx8 if self.mx else ra.rcclAmdStateF32, **args)

    def untouched(self, before):
        """Everything outside the tensors is as it was."""
        for b, old in zip(self.bufs, before):
            mask = np.ones(b.numel(), dtype=bool)
            for i in range(len(self.sizes)):
                if b is self.ms or b is self.vs:
                    mask[self.sstarts[i]:self.sstarts[i] - (-self.sizes[i] // 32)] = False
                else:
                    mask[self.starts[i]:self.starts[i] + self.sizes[i]] = False
            if b is self.grad:
                mask[:] = True
            a, o = (x.view(self.torch.uint8).view(x.numel(), -1).cpu().numpy() for x in (b, old))
            assert np.array_equal(a[mask], o[mask])


def _check_f32(case, before, coef, **hyper):
    """Every tensor of an fp32-state call against the formulas in 64 bits."""
    h = dict(HYPER, **hyper)
    pt, _, ct = case.names
    old = {id(b): o for b, o in zip(case.bufs, before)}
    for i in range(len(case.sizes)):
        p0, g0, m0, v0 = (_np(case.cut(old[id(b)], i)) for b in (case.param, case.grad, case.m, case.v))
        p, m, v, ep, em, ev = ref.adamw64(p0, g0, m0, v0, coef=coef, **{k: h[k] for k in ("lr", "beta1", "beta2", "eps", "weight_decay", "step")})
        assert np.all(np.abs(_np(case.cut(case.m, i)) - m) <= em), (case.sizes[i], "m")
        assert np.all(np.abs(_np(case.cut(case.v, i)) - v) <= ev), (case.sizes[i], "v")
        for buf, kind in ((case.param, pt), (case.copy, ct)):
            if buf is None:
                continue
            half = 0.0 if kind == "f32" else ref.HALF_STEP[kind]                  # rounding p to its type: half a step of it
            bound = ep + half * (np.abs(p) + ep) + ref.TINY[kind] / 2
            assert np.all(np.abs(_np(case.cut(buf, i)) - p) <= bound), (case.sizes[i], kind)
    case.untouched(before)


@pytest.mark.parametrize("param", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("grad", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("copy", [None, "f32", "bf16", "f16"])
def test_adamw_fp32_states(param, grad, copy):
    case = Case(SIZES, param, grad, copy, shift=0)
    before = case.snapshot()
    case.run(grad_scale=0.5)
    _check_f32(case, before, 0.5)


@pytest.mark.parametrize("shift", [1, 2, 3, 5])
@pytest.mark.parametrize("param,grad", [("f32", "bf16"), ("bf16", "f32"), ("f16", "f16")])
def test_adamw_views_at_any_element(shift, param, grad):
    case = Case(SIZES, param, grad, "bf16", shift=shift, seed=shift)
    before = case.snapshot()
    case.run()
    _check_f32(case, before, 1.0)


@pytest.mark.parametrize("kind", ["zero gradient", "zero state", "tiny", "huge", "first step"])
def test_adamw_values_at_the_edges(kind):
    case = Case([1000], "f32", "f32", None, seed=3)
    kw = {}
    if kind == "zero gradient":
        case.grad.zero_()
    elif kind == "zero state":
        case.m.zero_(), case.v.zero_(), case.grad[::2].zero_()            # 0 / (0 + eps) is 0
    elif kind == "tiny":
        case.grad.mul_(1e-18), case.m.mul_(1e-18), case.v.mul_(1e-36)
    elif kind == "huge":
        case.grad.mul_(1e18), case.m.mul_(1e18), case.v.mul_(1e36)
    else:
        case.m.zero_(), case.v.zero_()
        kw = dict(step=1)
    before = case.snapshot()
    case.run(**kw)
    _check_f32(case, before, 1.0, **kw)


def test_many_tensors_take_several_launches():
    """300 tensors, empty ones among them: what a call fits into one launch is less."""
    rng = np.random.default_rng(5)
    sizes = [int(x) for x in rng.integers(0, 400, 300)]
    sizes[0] = sizes[150] = sizes[299] = 0
    case = Case(sizes, "f32", "bf16", "bf16", seed=6)
    before = case.snapshot()
    case.run()
    _check_f32(case, before, 1.0)


def test_non_finite_gradients_stay_in_their_elements():
    import torch
    case = Case([1000], "f32", "f32", None)
    g = case.cut(case.grad, 0)
    g[10], g[500], g[999] = float("nan"), float("inf"), float("-inf")
    keep = torch.ones(1000, dtype=torch.bool)
    keep[[10, 500, 999]] = False
    before = case.snapshot()
    case.run()
    p, m = case.cut(case.param, 0).cpu(), case.cut(case.m, 0).cpu()
    assert not torch.isfinite(p[~keep]).any() and not torch.isfinite(m[~keep]).any()
    assert torch.isfinite(p[keep]).all()
    for b, old in zip(case.bufs, before):                                  # and the others are those of the clean formula
        b[case.starts[0] + np.array([10, 500, 999])] = old[case.starts[0] + np.array([10, 500, 999])]
    clean = Case([1000], "f32", "f32", None)
    clean.run()
    for a, b in ((case.param, clean.param), (case.m, clean.m), (case.v, clean.v)):
        assert torch.equal(case.cut(a, 0).cpu()[keep], clean.cut(b, 0).cpu()[keep])


# ------------------------------------------------------------------ 8-bit states
def _f32(x):
    return np.asarray(x, dtype=np.float32)


def _mx_expect(case, before, coef, seed, **hyper):
    """The kernel's arithmetic, rounding by rounding in fp32, then the rounding to 8 bits from its definition."""
    h = dict(HYPER, **hyper)
    old = {id(b): o for b, o in zip(case.bufs, before)}
    f = np.float32
    out = []
    for i, n in enumerate(case.sizes):
        p0, g0 = (case.cut(old[id(b)], i).float().cpu().numpy() for b in (case.param, case.grad))
        cm, cv = (_np(case.cut(old[id(b)], i)) for b in (case.m, case.v))
        sm, sv = (_np(case.cut_scale(old[id(b)], i)) for b in (case.ms, case.vs))
        m0, r0 = _f32(ref.mx_decode(cm, sm)), _f32(ref.mx_decode(cv, sv))
        g = g0 * f(coef)
        m = f(h["beta1"]) * m0 + f(1 - h["beta1"]) * g
        v = f(h["beta2"]) * (r0 * r0) + f(1 - h["beta2"]) * (g * g)
        r = np.sqrt(v)
        p = p0 * f(1 - h["lr"] * h["weight_decay"]) - f(h["lr"] / (1 - h["beta1"] ** h["step"])) * (m / (r * f(1 / math.sqrt(1 - h["beta2"] ** h["step"])) + f(h["eps"])))
        bits = ref.hash32(seed, h["step"], i, np.arange(n, dtype=np.uint64))
        # the update may be a product with a reciprocal that is off by one unit of its last place (2^-23 of it): two roundings
        # more than the quotient here, one of the product with the step size and one of the difference
        upd = np.abs(h["lr"] / (1 - h["beta1"] ** h["step"]) * m / (r / math.sqrt(1 - h["beta2"] ** h["step"]) + h["eps"]))
        slack = 1.01 * ref.U * (2 * 5 * upd + 2 * np.abs(p)) + 2.0 ** -148
        out.append(((p, slack), ref.mx_encode(m, (bits & np.uint64(0xFFFF)).astype(np.int64), False), ref.mx_encode(r, (bits >> np.uint64(16)).astype(np.int64), True)))
    return out


def _check_mx(case, before, coef, seed, **hyper):
    torch = case.torch
    for i, ((p, slack), (cm, sm), (cv, sv)) in enumerate(_mx_expect(case, before, coef, seed, **hyper)):
        assert np.array_equal(_np(case.cut_scale(case.ms, i)), sm) and np.array_equal(_np(case.cut_scale(case.vs, i)), sv), case.sizes[i]
        # (a negative value that is rounded to zero keeps its sign)
        assert np.array_equal(_np(case.cut(case.m, i)), cm), (case.sizes[i], "m")
        assert np.array_equal(_np(case.cut(case.v, i)), cv), (case.sizes[i], "sqrt v")
        for buf in (case.param, case.copy):
            if buf is not None:
                kind = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}[buf.dtype]
                half = 0.0 if kind == "f32" else ref.HALF_STEP[kind]
                p64 = p.astype(np.float64)
                assert np.all(np.abs(_np(case.cut(buf, i)) - p64) <= slack + half * (np.abs(p64) + slack) + ref.TINY[kind] / 2), (case.sizes[i], buf.dtype)
    case.untouched(before)


@pytest.mark.parametrize("param,grad,copy", [("f32", "bf16", "bf16"), ("f32", "f32", None), ("bf16", "bf16", None), ("f16", "f16", "f32"), ("bf16", "f32", "f16"),
                                             ("f16", "bf16", None), ("f32", "f16", "f16"), ("bf16", "f16", None), ("f16", "f32", "bf16")])
@pytest.mark.parametrize("shift", [0, 3])
def test_adamw_8_bit_states(param, grad, copy, shift):
    case = Case(SIZES, param, grad, copy, mx=True, shift=shift, seed=11, scale=1e-4)
    before = case.snapshot()
    case.run(seed=0x1234567890ABCDEF, grad_scale=0.25)
    _check_mx(case, before, 0.25, 0x1234567890ABCDEF)


def test_8_bit_states_from_zero_and_over_wide_blocks():
    """The first step from zeroed states; blocks whose values span many powers of two, zeros and whole zero blocks."""
    case = Case([4096, 100], "f32", "f32", None, mx=True, seed=12)
    for b in (case.m, case.v, case.ms, case.vs):
        b.zero_()
    case.grad.mul_(case.torch.exp2(case.torch.arange(case.grad.numel(), device="cuda") % 37 - 30.0))
    case.grad[::5] = 0
    case.cut(case.grad, 0)[64:128] = 0
    for step in (1, 2, 3):
        before = case.snapshot()
        case.run(step=step, seed=99)
        _check_mx(case, before, 1.0, 99, step=step)
    assert not _np(case.cut(case.m, 0))[64:128].any()


def test_8_bit_second_moment_never_freezes():
    """Without gradients sqrt(v) decays by sqrt(beta2) in each step: 65536 equal elements, 200 steps with beta2 = 0.99, each
    far below half a step of the 8-bit grid.  One rounding moves an element by at most an eighth of its value; the errors of
    the steps shrink with the value itself, so the relative variance of the end is at most 200 * (1/8)^2 * 1/4 (a rounding
    up with probability q has variance q (1 - q) <= 1/4) = 0.78, and the mean of 65536 elements is within 6 sigma = 0.021."""
    import rccl_amd as ra
    case = Case([65536], "f32", "f32", None, mx=True)
    case.grad.zero_()
    case.m.zero_()
    case.v.fill_(0x78)                 # 256 = 2^8, in the upper half of the grid
    case.vs.fill_(110)
    case.param.zero_()
    table = case.table()
    for step in range(1, 201):
        ra.adamw(table, ra.ncclFloat32, ra.ncclFloat32, -1, ra.rcclAmdStateMx8, lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, step=step, seed=5)
    r = ref.mx_decode(_np(case.cut(case.v, 0)), _np(case.cut_scale(case.vs, 0)))
    want = 256 * 2.0 ** (110 - 127) * 0.99 ** 100
    assert abs(r.mean() / want - 1) < 0.021


def test_8_bit_rounding_is_unbiased():
    """The mean over 400 seeds of a state that is rounded: within 6 standard errors, as a rounding's deviation is at most half
    the distance of its neighbours."""
    import rccl_amd as ra
    n = 256
    case = Case([n], "f32", "f32", None, mx=True, seed=21)
    for b in (case.m, case.v, case.ms, case.vs):
        b.zero_()
    saved = [b.clone() for b in case.bufs]
    total, gap = np.zeros(n), None
    table = case.table()
    for seed in range(400):
        for b, s in zip(case.bufs, saved):
            b.copy_(s)
        ra.adamw(table, ra.ncclFloat32, ra.ncclFloat32, -1, ra.rcclAmdStateMx8, lr=0.0, beta1=0.5, beta2=0.5, step=1, weight_decay=0.0, seed=seed * 0x9E3779B97F4A7C15 % 2 ** 64)
        total += ref.mx_decode(_np(case.cut(case.m, 0)), _np(case.cut_scale(case.ms, 0)))
    want = 0.5 * _np(case.cut(case.grad, 0))
    unit = 2.0 ** (_np(case.cut_scale(case.ms, 0)).astype(np.float64) - 127).repeat(32)
    y = np.abs(want) / unit
    gap = np.maximum(2.0 ** -9, 2.0 ** (np.floor(np.log2(np.maximum(y, 1e-30))) - 3)) * unit
    assert np.all(np.abs(total / 400 - want) <= 6 * 0.5 * gap / math.sqrt(400) + 1e-12)


def test_8_bit_non_finite_gradients():
    """An element whose moment is not finite becomes NaN; the others of its block are rounded as if it were not there."""
    case = Case([256, 40], "f32", "f32", None, mx=True, seed=22, scale=1e-4)
    for i, k, v in ((0, 40, "inf"), (0, 200, "nan"), (0, 201, "-inf"), (1, 39, "nan")):
        case.cut(case.grad, i)[k] = float(v)
    case.cut(case.grad, 0)[96:128] = float("inf")               # a block with nothing finite
    before = case.snapshot()
    case.run(seed=1)
    with np.errstate(all="ignore"):
        want = _mx_expect(case, before, 1.0, 1)
    for i, (_, (cm, sm), (cv, sv)) in enumerate(want):
        assert np.array_equal(_np(case.cut_scale(case.ms, i)), sm) and np.array_equal(_np(case.cut_scale(case.vs, i)), sv)
        for buf, code in ((case.m, cm), (case.v, cv)):
            got, bad = _np(case.cut(buf, i)), (code & 0x7F) == 0x7F
            assert bad.sum() == (35 if i == 0 else 1) and np.all((got[bad] & 0x7F) == 0x7F)
            assert np.array_equal(got[~bad], code[~bad])
    assert np.isfinite(_np(case.cut(case.param, 0))).sum() == 256 - 35


def test_8_bit_states_past_32_bits_of_elements():
    """One tensor of 2^32 + 1000 elements: the last elements against the definition (the hash takes the high word in)."""
    import torch
    import rccl_amd as ra
    n = 2 ** 32 + 1000
    if torch.cuda.mem_get_info()[0] < 40 * 2 ** 30:
        pytest.skip("needs 40 GiB of free device memory")
    p, g = (torch.zeros(n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2))
    ms, vs = (torch.zeros(-(-n // 32), dtype=torch.uint8, device="cuda") for _ in range(2))
    tail = 2048                                          # from 2^32 - 1048 on: both sides of the border
    at = n - tail
    at -= at % 32
    rng = np.random.default_rng(1)
    g[at:] = torch.from_numpy(rng.standard_normal(n - at).astype(np.float32)).to(torch.bfloat16).cuda()
    g[:4096] = g[at:at + 1]
    ra.adamw(np.array([ra.adamw_tensor(p, g, m, v, exp_avg_scale=ms, exp_avg_sq_scale=vs)]), ra.ncclBfloat16, ra.ncclBfloat16, -1, ra.rcclAmdStateMx8,
             lr=1e-2, beta1=0.5, beta2=0.5, eps=1e-8, weight_decay=0.0, step=1, seed=77)
    gg = g[at:].float().cpu().numpy()
    mm, rr = np.float32(0.5) * gg, np.sqrt(np.float32(0.5) * (gg * gg))
    bits = ref.hash32(77, 1, 0, np.arange(at, n, dtype=np.uint64))
    cm, sm = ref.mx_encode(mm, (bits & np.uint64(0xFFFF)).astype(np.int64), False)
    cv, sv = ref.mx_encode(rr, (bits >> np.uint64(16)).astype(np.int64), True)
    assert np.array_equal(m[at:].cpu().numpy(), cm) and np.array_equal(ms[at // 32:].cpu().numpy(), sm)
    assert np.array_equal(v[at:].cpu().numpy(), cv) and np.array_equal(vs[at // 32:].cpu().numpy(), sv)
    assert not m[4096:at].any() and not p[4096:at].any()


def test_8_bit_states_at_every_scale_byte():
    """Every code with every scale byte X is the code's value times 2^(X-127), as an fp32 number (past its largest: infinite),
    and NaN where X is 255.  With p = 0, no gradient, v = 0, eps = 1, beta1 = lr = 0.5 the step is p = -m0 / 2: of halvings and
    products with 1, all exact but for the reciprocal of 1, which may be off by one unit of its last place (2^-23 of the value)."""
    import torch
    case = Case([65536], "f32", "f32", None, mx=True)
    case.grad.zero_(), case.param.zero_(), case.v.zero_(), case.vs.zero_()
    code = np.tile(np.arange(256, dtype=np.uint8), 256)
    scale = np.repeat(np.arange(256, dtype=np.uint8), 8)
    case.cut(case.m, 0).copy_(torch.from_numpy(code).cuda())
    case.cut_scale(case.ms, 0).copy_(torch.from_numpy(scale).cuda())
    before = case.snapshot()
    case.run(lr=0.5, beta1=0.5, beta2=0.5, eps=1.0, weight_decay=0.0, step=1, seed=9)
    with np.errstate(all="ignore"):
        m0 = (ref.E4M3[code] * 2.0 ** (np.repeat(scale, 32).astype(np.float64) - 127)).astype(np.float32)
        m0[np.repeat(scale, 32) == 255] = np.nan
        m = np.float32(0.5) * m0 + np.float32(0.0)                 # (-0 + 0 is 0)
    p = _np(case.cut(case.param, 0))
    fine = np.isfinite(m)
    assert np.array_equal(np.isnan(p), np.isnan(m)) and np.array_equal(p[np.isinf(m)], -m[np.isinf(m)].astype(np.float64))
    assert np.all(np.abs(p[fine] + m[fine]) <= 2.0 ** -23 * np.abs(m[fine].astype(np.float64)) + 2.0 ** -149 * (np.abs(m[fine]) < 2.0 ** -126))
    bits = ref.hash32(9, 1, 0, np.arange(code.size, dtype=np.uint64))
    want, new = ref.mx_encode(m, (bits & np.uint64(0xFFFF)).astype(np.int64), False)
    got = _np(case.cut(case.m, 0))
    assert np.array_equal(_np(case.cut_scale(case.ms, 0)), new)
    assert np.array_equal(got[fine], want[fine]) and np.all((got[~fine] & 0x7F) == 0x7F)
    assert not _np(case.cut(case.v, 0)).any()
    case.untouched(before)


@pytest.mark.parametrize("eps", [0.0, 2.0 ** -126, 1e-30, 2.0 ** -75, 1.0, 2.0 ** 126])
def test_8_bit_states_divided_by_eps_alone(eps):
    """The divisor is eps, from one end of its range to the other: gradients whose squares vanish in fp32, or are next to
    nothing beside 2^126 (and large enough for the quotient to be a normal number)."""
    case = Case([5000], "f32", "f32", None, mx=True, seed=23)
    case.grad.mul_(1e-22), case.param.zero_()
    case.cut(case.grad, 0)[::7] = 0
    for b in (case.m, case.v, case.ms, case.vs):
        b.zero_()
    if eps == 2.0 ** 126:
        case.grad.mul_(1e38).clamp_(-1e16, 1e16)
    before = case.snapshot()
    case.run(eps=eps, step=1, seed=6)
    if eps == 0.0:
        g, p = case.cut(case.grad, 0), case.cut(case.param, 0)
        assert (p[g > 0] == -float("inf")).all() and (p[g < 0] == float("inf")).all() and p[g == 0].isnan().all()
        return
    _check_mx(case, before, 1.0, 6, eps=eps, step=1)


# ------------------------------------------------------------------ norm, clipping, skipping, device scalars
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shift", [0, 1])
def test_sum_squares(dtype, shift):
    import torch
    import rccl_amd as ra
    kind, tt = _types()[dtype]
    rng = np.random.default_rng(2)
    out = torch.full((1,), 123.0, dtype=torch.float64, device="cuda")
    for sizes in ([0], [1], [5], [4096], [4097], [3, 0, 70001, 1], [int(x) for x in rng.integers(0, 3000, 600)], [20_000_003]):
        flat = torch.from_numpy(rng.standard_normal(sum(sizes) + shift).astype(np.float32)).to(tt).cuda()
        tensors, at = [], shift
        for n in sizes:
            tensors.append(flat[at:at + n])
            at += n
        work = torch.empty(ra.sum_squares_bytes(len(sizes)), dtype=torch.uint8, device="cuda")
        ra.sum_squares(tensors, None, kind, out, work)
        x = flat[shift:].double().cpu().numpy()
        want = math.fsum(x * x)                        # squares of 24-bit numbers are exact in 64 bits
        # at most 2^14 additions to one partial sum, of positive terms, and some 30 to join them
        assert abs(float(out) - want) <= (2 ** 14 + 30) * 2.0 ** -53 * want, sizes[:4]
        first = float(out)
        ra.sum_squares(tensors, None, kind, out, work)
        assert float(out) == first                     # the same bits again
        ra.sum_squares(tensors, None, kind, out, work, accumulate=True)
        assert float(out) == first + first


def test_sum_squares_of_no_tensors_is_zero():
    import torch
    import rccl_amd as ra
    out = torch.full((1,), 7.0, dtype=torch.float64, device="cuda")
    ra.sum_squares([], None, ra.ncclBfloat16, out, None, accumulate=True)
    assert float(out) == 7.0
    ra.sum_squares([], None, ra.ncclBfloat16, out, None)
    assert float(out) == 0.0


def test_sum_squares_past_32_bits_of_elements():
    import torch
    import rccl_amd as ra
    n = 2 ** 32 + 2 ** 31 + 5
    if torch.cuda.mem_get_info()[0] < 20 * 2 ** 30:
        pytest.skip("needs 20 GiB of free device memory")
    x = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    for i, v in ((0, 1.0), (2 ** 31 - 1, 2.0), (2 ** 31, 3.0), (2 ** 32 - 1, 4.0), (2 ** 32, 5.0), (2 ** 32 + 2 ** 31, 6.0), (n - 1, 7.0)):
        x[i] = v
    out = torch.zeros(1, dtype=torch.float64, device="cuda")
    work = torch.empty(ra.sum_squares_bytes(2), dtype=torch.uint8, device="cuda")
    ra.sum_squares([x, x[:0]], None, ra.ncclBfloat16, out, work)
    assert float(out) == 1 + 4 + 9 + 16 + 25 + 36 + 49


def test_sum_squares_of_large_values_does_not_overflow():
    import torch
    import rccl_amd as ra
    x = torch.full((1000,), 1e30, dtype=torch.float32, device="cuda")
    out = torch.zeros(1, dtype=torch.float64, device="cuda")
    work = torch.empty(ra.sum_squares_bytes(1), dtype=torch.uint8, device="cuda")
    ra.sum_squares([x], None, ra.ncclFloat32, out, work)
    assert abs(float(out) / (1000 * float(np.float32(1e30)) ** 2) - 1) < 1e-12
    x[500] = float("inf")
    ra.sum_squares([x], None, ra.ncclFloat32, out, work)
    assert math.isinf(float(out))
    x[501] = float("nan")
    ra.sum_squares([x], None, ra.ncclFloat32, out, work)
    assert math.isnan(float(out))


@pytest.mark.parametrize("mx", [False, True])
def test_clipping_by_the_global_norm(mx):
    import torch
    import rccl_amd as ra
    case = Case(SIZES, "f32", "f32", "bf16", mx=mx, seed=31, scale=1e-4 if mx else 1e-2)
    out = torch.zeros(1, dtype=torch.float64, device="cuda")
    work = torch.empty(ra.sum_squares_bytes(len(SIZES)), dtype=torch.uint8, device="cuda")
    ra.sum_squares([case.cut(case.grad, i) for i in range(len(SIZES))], None, ra.ncclFloat32, out, work)
    norm = math.sqrt(float(out))
    for max_norm in (1e9, 0.25 * norm, 0.0):
        before = case.snapshot()
        coef = 0.5 * min(1.0, max_norm / (0.5 * norm + 1e-6))
        case.run(grad_scale=0.5, sum_sq=out, max_norm=max_norm, seed=3)
        if mx:
            _check_mx(case, before, coef, 3)
        else:
            _check_f32(case, before, coef)


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_norm_that_is_not_finite_skips_the_step(mx, bad):
    import torch
    case = Case(SIZES, "f32", "bf16", "bf16", mx=mx, seed=32)
    before = case.snapshot()
    case.run(sum_sq=torch.tensor([bad], dtype=torch.float64, device="cuda"), max_norm=1.0)
    for b, old in zip(case.bufs, before):
        if b is not case.copy:
            assert torch.equal(b.view(torch.uint8), old.view(torch.uint8))
    for i in range(len(SIZES)):
        assert torch.equal(case.cut(case.copy, i), case.cut(case.param, i).to(torch.bfloat16))
    case.untouched(before)


@pytest.mark.parametrize("mx", [False, True])
def test_step_and_rate_from_the_device(mx):
    """The kernel's own bias corrections against those of the host."""
    import torch
    for step in (1, 2, 1000, 123457):
        a, b = (Case(SIZES, "f32", "f32", None, mx=mx, seed=33) for _ in range(2))
        old = a.param.double()
        a.run(step=step, lr=float(np.float32(3e-3)), seed=4)
        b.run(step=1, lr=123.0, step_ptr=torch.tensor([step], dtype=torch.int64, device="cuda"),
              lr_ptr=torch.tensor([3e-3], dtype=torch.float32, device="cuda"), seed=4)
        for x, y in zip(a.bufs, b.bufs):
            if x.dtype == torch.uint8:
                assert torch.equal(x, y)
            elif x is a.param:     # constants that differ by a rounding: the update, at most |new| + |old|, by a few
                assert torch.all((x.double() - y.double()).abs() <= 8 * ref.U * (x.double().abs() + old.abs()))
            else:
                assert torch.equal(x, y)


def test_step_number_below_one_counts_as_one():
    import torch
    a, b = (Case([100], "f32", "f32", None, seed=36) for _ in range(2))
    a.run(step=1)
    b.run(step_ptr=torch.tensor([-3], dtype=torch.int64, device="cuda"))
    assert torch.equal(a.param, b.param)


@pytest.mark.parametrize("layout", ["flat", "scattered", "mixed copies", "reversed"])
@pytest.mark.parametrize("mx", [False, True])
def test_layouts_of_many_tensors(layout, mx):
    """Tensors that lie alike in flat buffers take one kind of launch, any others another: the results are the same bits."""
    import torch
    import rccl_amd as ra
    rng = np.random.default_rng(7)
    sizes = [int(x) for x in rng.integers(0, 300, 400)]
    a, b = (Case(sizes, "f32", "bf16", "bf16", mx=mx, seed=37) for _ in range(2))
    ty = _types()

    def run(case, table):
        ra.adamw(table, ty["f32"][0], ty["bf16"][0], ty["bf16"][0], ra.rcclAmdStateMx8 if mx else ra.rcclAmdStateF32, seed=5, **HYPER)

    ta, tb = a.table(), b.table()
    run(a, ta)
    order = np.arange(len(sizes))
    keep = []
    if layout == "scattered":                       # one gradient of a tensor lies elsewhere
        i = next(i for i in range(100, 400) if sizes[i] > 10)
        keep.append(b.cut(b.grad, i).clone())
        tb[i, 1] = keep[0].data_ptr()
    elif layout == "mixed copies":
        skip = [i for i in range(len(sizes)) if i % 3 == 0]
        tb[skip, 6] = 0
        for i in skip:
            b.cut(b.copy, i).copy_(a.cut(a.copy, i))
    elif layout == "reversed":                      # (the place of a tensor in the call is part of its random bits)
        order = order[::-1]
        if mx:
            tb = tb[order]
            before = b.snapshot()
            run(b, tb)
            f = [order.tolist().index(i) for i in range(len(sizes))]
            for i in range(0, len(sizes), 37):
                n = sizes[i]
                old = {id(x): o for x, o in zip(b.bufs, before)}
                g = b.cut(b.grad, i).float().cpu().numpy()
                m0 = _f32(ref.mx_decode(_np(b.cut(old[id(b.m)], i)), _np(b.cut_scale(old[id(b.ms)], i))))
                m = np.float32(HYPER["beta1"]) * m0 + np.float32(1 - HYPER["beta1"]) * g
                bits = ref.hash32(5, HYPER["step"], f[i], np.arange(n, dtype=np.uint64))
                code, scale = ref.mx_encode(m, (bits & np.uint64(0xFFFF)).astype(np.int64), False)
                assert np.array_equal(_np(b.cut(b.m, i)), code) and np.array_equal(_np(b.cut_scale(b.ms, i)), scale)
            return
    run(b, tb[order])
    for x, y in zip(a.bufs, b.bufs):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), layout


@pytest.mark.parametrize("mx", [False, True])
def test_captured_step_replays(mx):
    """sum of squares and AdamW in a graph, the step number and the rate on the device: each replay is the eager step."""
    import torch
    import rccl_amd as ra
    a, b = (Case([1000, 33, 5000], "f32", "bf16", "bf16", mx=mx, seed=34) for _ in range(2))
    step = torch.tensor([1], dtype=torch.int64, device="cuda")
    rate = torch.tensor([1e-2], dtype=torch.float32, device="cuda")
    outs = [torch.zeros(1, dtype=torch.float64, device="cuda") for _ in range(2)]
    works = [torch.empty(ra.sum_squares_bytes(3), dtype=torch.uint8, device="cuda") for _ in range(2)]
    kind = ra.ncclBfloat16

    def one(case, out, work):
        ra.sum_squares([case.cut(case.grad, i) for i in range(3)], None, kind, out, work)
        case.run(step_ptr=step, lr_ptr=rate, sum_sq=out, max_norm=0.1, seed=8)

    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        one(b, outs[1], works[1])
    for k in range(4):
        step.fill_(k + 1)
        rate.fill_(1e-2 / (k + 1))
        grad = torch.randn(a.grad.numel(), device="cuda").to(torch.bfloat16)
        a.grad.copy_(grad), b.grad.copy_(grad)
        one(a, outs[0], works[0])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(a.bufs, b.bufs):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), k
        assert float(outs[0]) == float(outs[1])


def test_on_another_stream():
    import torch
    a, b = (Case([100000], "f32", "bf16", "bf16", seed=35) for _ in range(2))
    a.run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    b.run(stream=s)
    s.synchronize()
    torch.cuda.synchronize()
    for x, y in zip(a.bufs, b.bufs):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_element_types_of_a_row():
    """Moments of the wrong size, or parameters that are not of the type adamw() will be given, would be read past their end."""
    import torch
    import rccl_amd as ra
    f, h = torch.zeros(64, device="cuda"), torch.zeros(64, dtype=torch.bfloat16, device="cuda")
    b, sc = torch.zeros(64, dtype=torch.uint8, device="cuda"), torch.zeros(2, dtype=torch.uint8, device="cuda")
    t = dict(param_type=ra.ncclFloat32, grad_type=ra.ncclBfloat16, copy_type=ra.ncclFloat16)
    assert ra.adamw_tensor(f, h, f, f, **t) == ra.adamw_tensor(f.data_ptr(), h, f, f, 64)
    assert ra.adamw_tensor(f, h, b, b, exp_avg_scale=sc, exp_avg_sq_scale=sc, copy=h.half(), **t)[7] == 64
    for call in (lambda: ra.adamw_tensor(f, f, b, f), lambda: ra.adamw_tensor(f, f, f, h), lambda: ra.adamw_tensor(f, f, f, f.int()),
                 lambda: ra.adamw_tensor(f, f, f, f, exp_avg_scale=sc, exp_avg_sq_scale=sc), lambda: ra.adamw_tensor(f, f, b, b, exp_avg_scale=sc.int(), exp_avg_sq_scale=sc),
                 lambda: ra.adamw_tensor(h, h, f, f, **t), lambda: ra.adamw_tensor(f, f, f, f, **t), lambda: ra.adamw_tensor(f, h, f, f, copy=f, **t)):
        with pytest.raises(ra.NcclError) as e:
            call()
        assert e.value.code == ra.ncclInvalidArgument


def test_an_older_error_is_not_reported_by_a_launch():
    """A call reports what its own launches say; the error that another call of the program left stays with the program."""
    import ctypes
    import torch
    hip = ctypes.CDLL(next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line))      # the one in use
    a, b = (Case([1000], "f32", "f32", None, seed=5) for _ in range(2))
    a.run()
    torch.cuda.synchronize()
    assert hip.hipSetDevice(1000) != 0                     # refused by the host, and remembered
    b.run()
    assert hip.hipGetLastError() != 0
    torch.cuda.synchronize()
    for x, y in zip(a.bufs, b.bufs):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_tensor_checks_of_the_python_mirror():
    """Tensors of another type, size or place are refused before an address is taken."""
    import torch
    import rccl_amd as ra
    p = torch.zeros(100, device="cuda")
    out = torch.zeros(1, dtype=torch.float64, device="cuda")
    work = torch.empty(ra.sum_squares_bytes(1), dtype=torch.uint8, device="cuda")
    for call in (lambda: ra.adamw_tensor(p, p[:50], p, p),
                 lambda: ra.adamw_tensor(p, p.cpu(), p, p),
                 lambda: ra.adamw_tensor(torch.zeros(10, 10, device="cuda").t()[1:], p, p, p),
                 lambda: ra.sum_squares([p.half()], None, ra.ncclFloat32, out, work),
                 lambda: ra.sum_squares([p], None, ra.ncclFloat32, out.float(), work),
                 lambda: ra.sum_squares([p], None, ra.ncclFloat32, out, work[:100]),
                 lambda: ra.sum_squares([p], [101], ra.ncclFloat32, out, work)):
        with pytest.raises(ra.NcclError) as e:
            call()
        assert e.value.code == ra.ncclInvalidArgument
