"""Token slots sorted by expert, rows dispatched and combined, and the gradients, against references in 64 bits.

Runs in the test runner's own process, which thereby opens the GPU; the name sorts behind test_gpu_fullsize, whose beds use
sixteen processes of their own."""
import numpy as np
import pytest

import local_ref as ref

pytestmark = pytest.mark.gpu


def _types():
    import torch
    import rccl_amd as ra
    return {"f32": (ra.ncclFloat32, torch.float32), "bf16": (ra.ncclBfloat16, torch.bfloat16), "f16": (ra.ncclFloat16, torch.float16)}


# ------------------------------------------------------------------ sort
def _run_sort(ids, first, n, align, wide):
    import torch
    import rccl_amd as ra
    tokens, topk = ids.shape
    g = 16                                               # guards behind and before every output
    rows = ra.expert_rows(tokens, topk, n, align)
    dev = torch.from_numpy(ids.astype(np.int64 if wide else np.int32)).cuda()
    outs = [torch.full((k + 2 * g,), -77, dtype=torch.int32, device="cuda") for k in (tokens * topk, rows, n + 1, n)]
    nbytes = ra.expert_sort_bytes(tokens, topk, n)
    work = torch.full((nbytes + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    cut = [o[g:o.numel() - g] for o in outs]
    ra.expert_sort(dev, ra.ncclInt64 if wide else ra.ncclInt32, tokens, topk, first, n, align, *cut, workspace=work[:nbytes] if nbytes else None)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.all(o[:g] == -77) and torch.all(o[o.numel() - g:] == -77)
    assert torch.all(work[nbytes:] == 0xA5)
    return [c.cpu().numpy() for c in cut]


def _ids(rng, tokens, topk, experts, kind):
    if kind == "one":                                    # all of them one expert
        return np.full((tokens, topk), experts - 1, dtype=np.int64)
    if kind == "padded":
        ids = rng.integers(0, experts, (tokens, topk))
        ids[rng.random(tokens) < 0.4] = -1
        return ids
    if kind == "skewed":                                 # and duplicates in a token
        return np.minimum((rng.exponential(0.1, (tokens, topk)) * experts).astype(np.int64), experts - 1)
    return rng.integers(0, experts, (tokens, topk))


@pytest.mark.parametrize("tokens", [0, 1, 2, 63, 64, 65, 127, 513, 1025, 4097, 8193, 70001])
@pytest.mark.parametrize("topk,experts,first,n,align", [(1, 1, 0, 1, 1), (2, 8, 0, 8, 16), (8, 128, 16, 16, 128), (6, 64, 0, 64, 1), (1, 1000, 0, 1000, 7), (3, 256, 255, 1, 100), (8, 255, 0, 255, 8)])
def test_sort(tokens, topk, experts, first, n, align):
    rng = np.random.default_rng(tokens * 31 + n)
    for i, kind in enumerate(("flat", "padded", "skewed", "one")):
        if tokens > 5000 and kind in ("flat",):
            continue
        ids = _ids(rng, tokens, topk, experts, kind)
        want = ref.expert_sort(ids, first, n, align)
        got = _run_sort(ids, first, n, align, wide=bool(i % 2))
        for name, a, b in zip(("position", "source", "offsets", "counts"), got, want):
            assert np.array_equal(a, b), (kind, name)


@pytest.mark.parametrize("tokens,topk,n", [(5, 64, 1024), (3000, 10, 1024), (1000, 33, 3)])
def test_sort_at_the_limits(tokens, topk, n):
    rng = np.random.default_rng(9)
    ids = _ids(rng, tokens, topk, n, "padded")
    for a, b in zip(_run_sort(ids, 0, n, 1024, True), ref.expert_sort(ids, 0, n, 1024)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("tokens,topk,n", [(65536, 8, 16), (65537, 8, 17), (65536, 8, 32), (65537, 8, 32), (65536, 8, 128), (65537, 8, 128), (131073, 2, 1024), (300001, 8, 4), (300001, 8, 17), (300001, 8, 300)])
def test_sort_at_tile_sizes(tokens, topk, n):
    """Tiles of each size, with the counts of all tiles added up by every tile or by a launch in between, at both sides of the limit."""
    ids = _ids(np.random.default_rng(tokens + n), tokens, topk, n, "padded")
    for a, b in zip(_run_sort(ids, 0, n, 8, True), ref.expert_sort(ids, 0, n, 8)):
        assert np.array_equal(a, b)


def test_sort_of_ids_that_are_far_out():
    """Ids outside every range, the extremes of int64 among them, are dropped."""
    ids = np.array([[-2 ** 63, 2 ** 63 - 1], [2 ** 32, 2 ** 32 + 5], [5, -1], [6, 4], [7, 5]], dtype=np.int64)
    for a, b in zip(_run_sort(ids, 5, 2, 4, True), ref.expert_sort(ids, 5, 2, 4)):
        assert np.array_equal(a, b)


def test_sort_without_the_optional_outputs():
    import torch
    import rccl_amd as ra
    ids = np.random.default_rng(3).integers(-1, 8, (50, 2))
    position = torch.empty(100, dtype=torch.int32, device="cuda")
    ra.expert_sort(torch.from_numpy(ids).cuda(), ra.ncclInt64, 50, 2, 0, 8, 4, position)
    assert np.array_equal(position.cpu().numpy(), ref.expert_sort(ids, 0, 8, 4)[0])


def test_sort_of_many_slots():
    """Four million slots of 128 experts: stable, complete and in range (checked by sorting)."""
    import torch
    import rccl_amd as ra
    tokens, topk, n = 500_009, 8, 128
    ids = torch.randint(-1, n, (tokens, topk), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    position = torch.empty(tokens * topk, dtype=torch.int32, device="cuda")
    source = torch.empty(ra.expert_rows(tokens, topk, n, 1), dtype=torch.int32, device="cuda")
    work = torch.empty(ra.expert_sort_bytes(tokens, topk, n), dtype=torch.uint8, device="cuda")
    ra.expert_sort(ids, ra.ncclInt64, tokens, topk, 0, n, 1, position, source, workspace=work)
    flat = ids.view(-1)
    key, order = torch.sort(torch.where(flat < 0, n, flat), stable=True)
    held = int((key < n).sum())
    assert torch.equal(source[:held].long(), order[:held]) and torch.all(source[held:] == -1)
    want = torch.full((tokens * topk,), -1, dtype=torch.int64, device="cuda")
    want[order[:held]] = torch.arange(held, device="cuda")
    assert torch.equal(position.long(), want)


# ------------------------------------------------------------------ rows
class Rows:
    """Routing, and matrices whose rows are `gap` elements further apart than they are long and begin `shift` elements into
    their storage, with guards on all sides."""

    def __init__(self, tokens, topk, hidden, dtype="bf16", n=8, align=4, gap=0, shift=0, seed=0, experts=None, kind="padded"):
        self.tokens, self.topk, self.hidden, self.n, self.gap, self.shift = tokens, topk, hidden, n, gap, shift
        self.rng = np.random.default_rng(seed)
        self.code, self.torch_type = _types()[dtype]
        self.dtype = dtype
        self.ids = _ids(self.rng, tokens, topk, experts or n, kind)
        self.position, self.source, self.offsets, self.counts = ref.expert_sort(self.ids, 0, n, align)
        self.rows = self.source.size
        self.dev = {}
        import torch
        for k in ("position", "offsets", "counts"):
            self.dev[k] = torch.from_numpy(getattr(self, k)).cuda()
        self.used = np.zeros(self.rows, dtype=bool)
        self.used[self.position[self.position >= 0]] = True
        self.pad = np.zeros(self.rows, dtype=bool)
        for e in range(n):
            self.pad[self.offsets[e] + self.counts[e]:self.offsets[e + 1]] = True

    def matrix(self, rows, fill=None):
        """(storage, view of `rows` rows); values of a normal distribution, or `fill`."""
        import torch
        wide = self.hidden + self.gap
        n = (rows + 2) * wide + self.shift + 16
        if fill is None:
            flat = torch.from_numpy(self.rng.standard_normal(n).astype(np.float32)).to(self.torch_type).cuda()
        else:
            flat = torch.full((n,), fill, dtype=self.torch_type, device="cuda")
        at = wide + self.shift
        return flat, flat[at:at + rows * wide].view(rows, wide)[:, :self.hidden] if rows else flat[at:at].view(0, wide)[:, :self.hidden]

    def weights(self, kind):
        import torch
        return torch.from_numpy(self.rng.standard_normal((self.tokens, self.topk)).astype(np.float32)).to(_types()[kind][1]).cuda()

    def slots(self):
        """position as (tokens, topk)."""
        return self.position.reshape(self.tokens, self.topk)


def _outside(flat, view, before):
    """What of the storage does not belong to the view is as it was."""
    import torch
    a, b = flat.clone(), before.clone()
    for t in (a, b):
        torch.as_strided(t, view.shape, view.stride(), view.storage_offset()).zero_()
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def _np64(t):
    return t.double().cpu().numpy()


ROWS = [(1, 1, 1, "bf16", 0, 0), (1, 8, 4096, "bf16", 0, 0), (3, 2, 7, "bf16", 1, 1), (65, 2, 8, "f16", 0, 0), (64, 3, 9, "f32", 3, 1), (130, 8, 63, "f16", 5, 3),
        (77, 6, 512, "bf16", 8, 0), (50, 64, 130, "bf16", 0, 2), (33, 4, 1000, "f32", 24, 0), (40, 5, 1001, "f32", 0, 0), (300, 2, 2048, "f16", 0, 0),
        (19, 8, 4097, "bf16", 7, 1), (9000, 4, 100, "bf16", 0, 1), (9000, 4, 70, "f32", 1, 0), (20001, 3, 129, "f16", 0, 0), (30000, 2, 5, "bf16", 0, 0), (9, 8, 8200, "f32", 0, 0), (5, 3, 33000, "bf16", 0, 0), (2000, 4, 16, "bf16", 0, 0)]


@pytest.mark.parametrize("tokens,topk,hidden,dtype,gap,shift", ROWS)
def test_dispatch(tokens, topk, hidden, dtype, gap, shift):
    import torch
    import rccl_amd as ra
    r = Rows(tokens, topk, hidden, dtype, gap=gap, shift=shift)
    _, x = r.matrix(tokens)
    x[tokens // 2, :] = float("nan")                   # moved like any value
    for padded in (True, False):
        flat, out = r.matrix(r.rows, 5.0)
        before = flat.clone()
        ra.expert_dispatch(x, out, r.rows, r.code, tokens, topk, hidden, r.dev["position"], **(dict(offsets=r.dev["offsets"], counts=r.dev["counts"], n_experts=r.n) if padded else {}))
        got, xs = _np64(out), _np64(x)
        want = np.full((r.rows, hidden), 5.0)
        for slot, row in enumerate(r.position):
            if row >= 0:
                want[row] = xs[slot // topk]
        if padded:
            want[r.pad] = 0.0
        assert np.array_equal(got, want, equal_nan=True)
        assert _outside(flat, out, before)


@pytest.mark.parametrize("tokens,topk,hidden,dtype,gap,shift", ROWS)
@pytest.mark.parametrize("weights", [None, "f32", "bf16", "f16"])
def test_combine(tokens, topk, hidden, dtype, gap, shift, weights):
    import rccl_amd as ra
    r = Rows(tokens, topk, hidden, dtype, gap=gap, shift=shift, seed=1)
    _, z = r.matrix(r.rows)
    z[np.flatnonzero(~r.used)] = float("nan")           # rows without a slot are never part of a sum
    w = r.weights(weights) if weights else None
    flat, y = r.matrix(tokens, 5.0)
    before = flat.clone()
    ra.expert_combine(z, r.rows, w, _types()[weights][0] if weights else -1, y, r.code, tokens, topk, hidden, r.dev["position"])
    zs, ws = _np64(z), _np64(w) if weights else np.ones((tokens, topk))
    want, size = np.zeros((tokens, hidden)), np.zeros((tokens, hidden))
    for k in range(topk):
        p = r.slots()[:, k]
        has = p >= 0
        want[has] += ws[has, k, None] * zs[p[has]]
        size[has] += np.abs(ws[has, k, None] * zs[p[has]])
    # one rounding in each of topk fused multiply-adds of sums that are at most `size`, and half a step of the type at the end
    bound = 1.01 * topk * ref.U * size
    bound += (ref.HALF_STEP[dtype] if dtype != "f32" else 0.0) * (np.abs(want) + bound) + ref.TINY[dtype]
    assert np.all(np.abs(_np64(y) - want) <= bound)
    assert _outside(flat, y, before)


@pytest.mark.parametrize("tokens,topk,hidden,dtype,gap,shift", ROWS)
@pytest.mark.parametrize("weights", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("in_place", [False, True])
def test_combine_backward(tokens, topk, hidden, dtype, gap, shift, weights, in_place):
    import torch
    import rccl_amd as ra
    r = Rows(tokens, topk, hidden, dtype, gap=gap, shift=shift, seed=2)
    _, dy = r.matrix(tokens)
    zflat, z = r.matrix(r.rows)
    z[np.flatnonzero(~r.used)] = float("nan")
    zs = _np64(z)
    w = r.weights(weights)
    dw = torch.full((tokens, topk), 9.0, dtype=w.dtype, device="cuda")
    flat, dz = (zflat, z) if in_place else r.matrix(r.rows, 5.0)
    before = flat.clone()
    ra.expert_combine_backward(dy, z, r.rows, w, _types()[weights][0], dz, dw, r.code, tokens, topk, hidden, r.dev["position"], r.dev["offsets"], r.dev["counts"], r.n)
    dys, ws = _np64(dy), _np64(w)
    want = zs.copy() if in_place else np.full((r.rows, hidden), 5.0)
    want_w, size = np.zeros((tokens, topk)), np.zeros((tokens, topk))
    for t in range(tokens):
        for k in range(topk):
            p = r.slots()[t, k]
            if p >= 0:
                want[p] = ws[t, k] * dys[t]
                want_w[t, k] = np.dot(dys[t], zs[p])
                size[t, k] = np.dot(np.abs(dys[t]), np.abs(zs[p]))
    want[r.pad] = 0.0
    # dz: one rounding in fp32, then half a step of the type.  A row that is behind the last expert is as it was.
    half = ref.HALF_STEP[dtype] if dtype != "f32" else 0.0
    bound = (1.01 * ref.U + half * 1.01) * np.abs(want) + ref.TINY[dtype]
    got = _np64(dz)
    keep = r.used | r.pad
    assert np.all(np.abs(got[keep] - want[keep]) <= bound[keep])
    assert np.array_equal(got[~keep], want[~keep], equal_nan=True)
    # dw: a lane adds the products of its part of the row (a 64th of it, in packs of at most 8 elements), then 6 sums join them
    halfw = ref.HALF_STEP[weights] if weights != "f32" else 0.0
    bound = 1.01 * (hidden // 64 + 8 + 6) * ref.U * size
    bound += halfw * (np.abs(want_w) + bound) + ref.TINY[weights]
    assert np.all(np.abs(_np64(dw) - want_w) <= bound)
    assert _outside(flat, dz, before)


@pytest.mark.parametrize("topk,tokens", [(8, 4500), (3, 11000), (1, 33000)])
@pytest.mark.parametrize("hidden,dtype,gap,shift", [(129, "f32", 0, 0), (257, "bf16", 0, 0), (400, "f16", 1, 3), (512, "bf16", 0, 0), (513, "bf16", 2, 1), (300, "f32", 1, 1),
                                                    (1023, "f16", 0, 5), (1024, "bf16", 8, 0), (1030, "bf16", 1, 0), (520, "f32", 0, 2), (2047, "bf16", 0, 0), (1024, "f32", 3, 0)])
def test_short_rows_of_many_slots(topk, tokens, hidden, dtype, gap, shift):
    """Rows of one to four KiB in so many slots that a wave takes several of them; a reference in 64 bits on the GPU."""
    import torch
    import rccl_amd as ra
    gen = torch.Generator("cuda").manual_seed(hidden + topk)
    code, tt = _types()[dtype]
    pos = torch.full((tokens * topk,), -1, dtype=torch.int64, device="cuda")
    keep = torch.rand(tokens * topk, device="cuda", generator=gen) < 0.9
    held = int(keep.sum())
    rows = held + 37                                    # the last ones belong to nobody
    pos[keep] = torch.randperm(held + 20, device="cuda", generator=gen)[:held]
    used = torch.zeros(rows, dtype=torch.bool, device="cuda")
    used[pos[keep]] = True
    pos32 = pos.to(torch.int32)
    wide = hidden + gap

    def matrix(r, fill=None):
        flat = torch.randn((r + 2) * wide + 64, device="cuda", generator=gen).to(tt) if fill is None else torch.full(((r + 2) * wide + 64,), fill, dtype=tt, device="cuda")
        return flat, flat[wide + shift:wide + shift + r * wide].view(r, wide)[:, :hidden]

    _, x = matrix(tokens)
    flat, out = matrix(rows, 5.0)
    before = flat.clone()
    ra.expert_dispatch(x, out, rows, code, tokens, topk, hidden, pos32)
    token = torch.arange(tokens * topk, device="cuda") // topk
    want = torch.full((rows, hidden), 5.0, dtype=tt, device="cuda")
    want[pos[keep]] = x[token[keep]]
    assert torch.equal(out, want) and _outside(flat, out, before)

    _, z = matrix(rows)
    z[~used] = float("nan")
    w = torch.randn(tokens, topk, device="cuda", generator=gen)
    flat, y = matrix(tokens, 5.0)
    before = flat.clone()
    ra.expert_combine(z, rows, w, ra.ncclFloat32, y, code, tokens, topk, hidden, pos32)
    zg = torch.where(keep[:, None], z[pos.clamp(min=0)].double(), 0.0).view(tokens, topk, hidden)
    terms = zg * w.double()[:, :, None]
    half = ref.HALF_STEP[dtype] if dtype != "f32" else 0.0
    bound = 1.01 * topk * ref.U * terms.abs().sum(1)
    bound += half * (terms.sum(1).abs() + bound) + ref.TINY[dtype]
    assert torch.all((y.double() - terms.sum(1)).abs() <= bound) and _outside(flat, y, before)

    _, dy = matrix(tokens)
    flat, dz = matrix(rows, 5.0)
    before = flat.clone()
    dw = torch.full((tokens, topk), 9.0, device="cuda")
    ra.expert_combine_backward(dy, z, rows, w, ra.ncclFloat32, dz, dw, code, tokens, topk, hidden, pos32)
    want = torch.full((rows, hidden), 5.0, dtype=torch.float64, device="cuda")
    want[pos[keep]] = dy[token[keep]].double() * w.double().view(-1)[keep, None]
    assert torch.all((dz.double() - want).abs() <= (1.01 * ref.U + 1.01 * half) * want.abs() + ref.TINY[dtype]) and _outside(flat, dz, before)
    prod = zg * dy.double()[:, None, :]
    assert torch.all((dw.double() - prod.sum(2)).abs() <= 1.01 * (hidden // 64 + 14) * ref.U * prod.abs().sum(2) + ref.TINY["f32"])


@pytest.mark.parametrize("hidden,dtype", [(512, "bf16"), (1000, "f16"), (1024, "f32"), (4104, "bf16")])
@pytest.mark.parametrize("n", [0, 1, 3, 6, 12, 24, 36, 64])
@pytest.mark.parametrize("how", ["offsets", "rows", "neither"])
def test_dropped_slots(hidden, dtype, n, how):
    """A rank that holds n of 64 experts (0: one that nobody chose): all, some or almost none of the slots are kept, which the
    offsets, the number of rows or only the positions say."""
    import torch
    import rccl_amd as ra
    gen = torch.Generator("cuda").manual_seed(hidden + n)
    code, tt = _types()[dtype]
    tokens, topk = 4500 if hidden < 2000 else 1100, 8
    ids = torch.randint(0, 64, (tokens, topk), device="cuda", generator=gen)
    n, first = (n, 0) if n else (1, 64)
    pos, off, cnt = (torch.empty(k, dtype=torch.int32, device="cuda") for k in (tokens * topk, n + 1, n))
    work = torch.empty(ra.expert_sort_bytes(tokens, topk, n), dtype=torch.uint8, device="cuda")
    ra.expert_sort(ids, ra.ncclInt64, tokens, topk, first, n, 4, pos, None, off, cnt, work)
    keep = pos >= 0
    assert torch.equal(keep, ((ids >= first) & (ids < first + n)).view(-1))
    held = int(off[-1])
    rows = held + 3 if how == "rows" else ra.expert_rows(tokens, topk, n, 4)
    segments = dict(offsets=off, counts=cnt, n_experts=n) if how == "offsets" else {}
    token = torch.arange(tokens * topk, device="cuda") // topk
    x, dy = (torch.randn(tokens, hidden, device="cuda", generator=gen).to(tt) for _ in range(2))
    z = torch.randn(rows, hidden, device="cuda", generator=gen).to(tt)
    w = torch.randn(tokens, topk, device="cuda", generator=gen)
    out, dz, dw = torch.full((rows, hidden), 5.0, dtype=tt, device="cuda"), torch.full((rows, hidden), 5.0, dtype=tt, device="cuda"), torch.full((tokens, topk), 9.0, device="cuda")
    ra.expert_dispatch(x, out, rows, code, tokens, topk, hidden, pos, **segments)
    ra.expert_combine_backward(dy, z, rows, w, ra.ncclFloat32, dz, dw, code, tokens, topk, hidden, pos, **segments)
    at = pos[keep].long()
    want, wantz = torch.full((rows, hidden), 5.0, dtype=tt, device="cuda"), torch.full((rows, hidden), 5.0, dtype=torch.float64, device="cuda")
    if how == "offsets":
        want[:held], wantz[:held] = 0.0, 0.0
    want[at] = x[token[keep]]
    assert torch.equal(out, want)
    half = ref.HALF_STEP[dtype] if dtype != "f32" else 0.0
    wantz[at] = dy[token[keep]].double() * w.view(-1)[keep, None].double()
    assert torch.all((dz.double() - wantz).abs() <= (1.01 * ref.U + 1.01 * half) * wantz.abs() + ref.TINY[dtype])
    prod = dy[token[keep]].double() * z[at].double()
    # a lane adds the products of its part of the row (a 64th of it, in packs of at most 8 elements), then 6 sums join them
    assert torch.all((dw.view(-1)[keep].double() - prod.sum(1)).abs() <= 1.01 * (hidden // 64 + 14) * ref.U * prod.abs().sum(1) + ref.TINY["f32"])
    assert torch.all(dw.view(-1)[~keep] == 0.0)


def test_gradients_against_differences():
    """<dy, combine(z, w)> is linear in z and in w: its differences are exact up to rounding, in fp32 with small whole numbers
    exactly.  The gradient of a dispatch is a combine without weights: <dout, dispatch(x)> = <combine(dout), x>."""
    import torch
    import rccl_amd as ra
    tokens, topk, hidden = 20, 3, 40
    r = Rows(tokens, topk, hidden, "f32", seed=4)
    whole = lambda *s: torch.from_numpy(r.rng.integers(-3, 4, s).astype(np.float32)).cuda()  # noqa: E731
    z, dy, w = whole(r.rows, hidden), whole(tokens, hidden), whole(tokens, topk)
    dz, dw = torch.zeros_like(z), torch.zeros_like(w)
    pos = r.dev["position"]

    def loss(z, w):
        y = torch.empty(tokens, hidden, device="cuda")
        ra.expert_combine(z, r.rows, w, ra.ncclFloat32, y, ra.ncclFloat32, tokens, topk, hidden, pos)
        return float((y.double() * dy.double()).sum())

    ra.expert_combine_backward(dy, z, r.rows, w, ra.ncclFloat32, dz, dw, ra.ncclFloat32, tokens, topk, hidden, pos, r.dev["offsets"], r.dev["counts"], r.n)
    base = loss(z, w)
    for _ in range(40):
        i, j = int(r.rng.integers(r.rows)), int(r.rng.integers(hidden))
        z2 = z.clone()
        z2[i, j] += 1
        assert loss(z2, w) - base == (float(dz[i, j]) if r.used[i] else 0.0)
        t, k = int(r.rng.integers(tokens)), int(r.rng.integers(topk))
        w2 = w.clone()
        w2[t, k] += 1
        assert loss(z, w2) - base == float(dw[t, k])
    x, dout = whole(tokens, hidden), whole(r.rows, hidden)
    out, dx = torch.zeros_like(dout), torch.empty_like(x)
    ra.expert_dispatch(x, out, r.rows, ra.ncclFloat32, tokens, topk, hidden, pos)
    ra.expert_combine(dout, r.rows, None, -1, dx, ra.ncclFloat32, tokens, topk, hidden, pos)
    assert float((out.double() * dout.double()).sum()) == float((dx.double() * x.double()).sum())


def test_positions_outside_the_rows_are_passed_over():
    """Positions of a larger order than the buffer has rows (and negative ones): nothing is read or written for them."""
    import torch
    import rccl_amd as ra
    tokens, topk, hidden, rows = 12, 2, 64, 6
    pos = np.array([0, 6, 5, -1, 2 ** 31 - 1, 1, -2 ** 31, 2, 100, 3, 7, 4] + [-1] * 12, dtype=np.int32)
    dev = torch.from_numpy(pos).cuda()
    x = torch.randn(tokens, hidden, device="cuda")
    flat = torch.full((rows + 20, hidden), 5.0, device="cuda")
    out = flat[:rows]
    ra.expert_dispatch(x, out, rows, ra.ncclFloat32, tokens, topk, hidden, dev)
    assert torch.all(flat[rows:] == 5.0)
    for slot, p in enumerate(pos):
        if 0 <= p < rows:
            assert torch.equal(out[p], x[slot // topk])
    y = torch.empty(tokens, hidden, device="cuda")
    ra.expert_combine(out, rows, None, -1, y, ra.ncclFloat32, tokens, topk, hidden, dev)
    for t in range(tokens):
        has = [p for p in pos[2 * t:2 * t + 2] if 0 <= p < rows]
        assert torch.equal(y[t], sum((out[p] for p in has), torch.zeros(hidden, device="cuda")))
    dz, dw = torch.zeros_like(flat), torch.full((tokens, topk), 9.0, device="cuda")
    ra.expert_combine_backward(x, out, rows, torch.ones(tokens, topk, device="cuda"), ra.ncclFloat32, dz, dw, ra.ncclFloat32, tokens, topk, hidden, dev)
    assert not dz[rows:].any()
    assert torch.equal(dw.view(-1) != 0, torch.from_numpy((pos >= 0) & (pos < rows)).cuda())


def test_large_rows_pass_32_bits_of_offset():
    """A buffer of more than 2^32 bytes: rows at its end."""
    import torch
    import rccl_amd as ra
    hidden, rows = 8192, 300_000                        # 4.9 GB of bf16
    if torch.cuda.mem_get_info()[0] < 16 * 2 ** 30:
        pytest.skip("needs 16 GiB of free device memory")
    tokens = 64
    pos = torch.arange(rows - tokens, rows, dtype=torch.int32, device="cuda")
    x = torch.randn(tokens, hidden, device="cuda").to(torch.bfloat16)
    out = torch.zeros(rows, hidden, dtype=torch.bfloat16, device="cuda")
    ra.expert_dispatch(x, out, rows, ra.ncclBfloat16, tokens, 1, hidden, pos)
    assert torch.equal(out[rows - tokens:], x) and not out[:rows - tokens].any()
    y = torch.empty_like(x)
    ra.expert_combine(out, rows, None, -1, y, ra.ncclBfloat16, tokens, 1, hidden, pos)
    assert torch.equal(y, x)
    w, dw = torch.full((tokens, 1), 2.0, device="cuda"), torch.empty(tokens, 1, device="cuda")
    ra.expert_combine_backward(x, out, rows, w, ra.ncclFloat32, out, dw, ra.ncclBfloat16, tokens, 1, hidden, pos)
    assert torch.equal(out[rows - tokens:], 2 * x)


def test_more_slots_than_a_launch_has_waves():
    """72 million slots of eight elements, moved by a permutation: a wave takes several slots."""
    import torch
    import rccl_amd as ra
    tokens, topk, hidden = 9_000_001, 8, 8
    rows = tokens * topk
    gen = torch.Generator("cuda").manual_seed(1)
    pos = torch.randperm(rows, device="cuda", generator=gen).to(torch.int32)
    x = torch.randint(-4, 5, (tokens, hidden), device="cuda", generator=gen).to(torch.bfloat16)
    out = torch.zeros(rows, hidden, dtype=torch.bfloat16, device="cuda")
    ra.expert_dispatch(x, out, rows, ra.ncclBfloat16, tokens, topk, hidden, pos)
    want = torch.empty_like(out)
    want[pos.long()] = x.repeat_interleave(topk, 0)
    assert torch.equal(out, want)
    y = torch.empty_like(x)
    ra.expert_combine(out, rows, None, -1, y, ra.ncclBfloat16, tokens, topk, hidden, pos)
    assert torch.equal(y, topk * x)
    w, dw = torch.full((tokens, topk), 2.0, device="cuda"), torch.empty(tokens, topk, device="cuda")
    ra.expert_combine_backward(x, out, rows, w, ra.ncclFloat32, out, dw, ra.ncclBfloat16, tokens, topk, hidden, pos)
    assert torch.equal(out, 2 * want)
    assert torch.equal(dw, x.float().square().sum(1, keepdim=True).expand(tokens, topk))


def test_no_tokens():
    import torch
    import rccl_amd as ra
    e = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    none = torch.empty(0, 2, dtype=torch.int32, device="cuda")
    out = torch.full((8, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    ra.expert_dispatch(e, out, 8, ra.ncclBfloat16, 0, 2, 64, none)
    ra.expert_combine(out, 8, None, -1, e, ra.ncclBfloat16, 0, 2, 64, none)
    w = torch.empty(0, 2, device="cuda")
    ra.expert_combine_backward(e, out, 8, w, ra.ncclFloat32, torch.empty_like(out), w.clone(), ra.ncclBfloat16, 0, 2, 64, none)
    assert torch.all(out == 5.0)
    # tokens, but no rows: everything is dropped
    y = torch.full((3, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    pos = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    ra.expert_combine(e, 0, None, -1, y, ra.ncclBfloat16, 3, 2, 64, pos)
    assert not y.any()


def test_captured_sort_and_rows_replay():
    """A layer's sort, dispatch, combine and backward in one graph: each replay with new routing is the eager result."""
    import torch
    import rccl_amd as ra
    tokens, topk, hidden, n, align = 3000, 4, 256, 16, 8
    rows = ra.expert_rows(tokens, topk, n, align)

    def buffers():
        i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        h = lambda r: torch.zeros(r, hidden, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        return dict(ids=torch.zeros(tokens, topk, dtype=torch.int64, device="cuda"), position=i(tokens, topk), source=i(rows), offsets=i(n + 1), counts=i(n),
                    work=torch.zeros(max(1, ra.expert_sort_bytes(tokens, topk, n)), dtype=torch.uint8, device="cuda"), x=h(tokens), out=h(rows), y=h(tokens), dz=h(rows),
                    w=torch.zeros(tokens, topk, device="cuda"), dw=torch.zeros(tokens, topk, device="cuda"))

    def layer(b):
        ra.expert_sort(b["ids"], ra.ncclInt64, tokens, topk, 0, n, align, b["position"], b["source"], b["offsets"], b["counts"], b["work"])
        seg = dict(offsets=b["offsets"], counts=b["counts"], n_experts=n)
        ra.expert_dispatch(b["x"], b["out"], rows, ra.ncclBfloat16, tokens, topk, hidden, b["position"], **seg)
        ra.expert_combine(b["out"], rows, b["w"], ra.ncclFloat32, b["y"], ra.ncclBfloat16, tokens, topk, hidden, b["position"])
        ra.expert_combine_backward(b["y"], b["out"], rows, b["w"], ra.ncclFloat32, b["dz"], b["dw"], ra.ncclBfloat16, tokens, topk, hidden, b["position"], **seg)

    a, b = buffers(), buffers()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        layer(b)
    gen = torch.Generator("cuda").manual_seed(3)
    for k in range(4):
        for key, new in (("ids", torch.randint(-1, n + k, (tokens, topk), device="cuda", generator=gen)), ("x", torch.randn(tokens, hidden, device="cuda", generator=gen)),
                         ("w", torch.rand(tokens, topk, device="cuda", generator=gen))):
            a[key].copy_(new), b[key].copy_(new)
        layer(a)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for key in a:
            assert torch.equal(a[key].view(torch.uint8), b[key].view(torch.uint8)), (k, key)


def test_device_pointers_and_streams_by_handle():
    """The same calls with addresses, strides and a stream handle in the place of tensors."""
    import torch
    import rccl_amd as ra
    r = Rows(50, 3, 100, "bf16", seed=6)
    (_, x), (_, out), (_, y), (_, dz) = r.matrix(50), r.matrix(r.rows, 0.0), r.matrix(50, 0.0), r.matrix(r.rows, 0.0)
    w, dw, ids = r.weights("f32"), torch.zeros(50, 3, device="cuda"), torch.from_numpy(r.ids.astype(np.int32)).cuda()
    pos, off, cnt = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (150, 9, 8))

    def run(at, stream, **strides):
        ra.expert_sort(at(ids), ra.ncclInt32, 50, 3, 0, 8, 4, at(pos), None, at(off), at(cnt), None, stream=stream)
        s = lambda *names: {n: v for n, v in strides.items() if n in names}  # noqa: E731
        ra.expert_dispatch(at(x), at(out), r.rows, r.code, 50, 3, 100, at(pos), at(off), at(cnt), 8, stream=stream, **s("x_stride", "out_stride"))
        ra.expert_combine(at(out), r.rows, at(w), ra.ncclFloat32, at(y), r.code, 50, 3, 100, at(pos), stream=stream, **s("z_stride", "y_stride"))
        ra.expert_combine_backward(at(y), at(out), r.rows, at(w), ra.ncclFloat32, at(dz), at(dw), r.code, 50, 3, 100, at(pos), stream=stream, **s("dy_stride", "z_stride", "dz_stride"))
        torch.cuda.synchronize()
        got = [t.clone() for t in (pos, off, cnt, out, y, dz, dw)]
        for t in (pos, off, cnt, out, y, dz, dw):
            t.zero_()
        torch.cuda.synchronize()
        return got

    st = torch.cuda.Stream()
    a = run(lambda t: t, None)
    b = run(lambda t: t.data_ptr(), st.cuda_stream, x_stride=100, out_stride=100, z_stride=100, y_stride=100, dy_stride=100, dz_stride=100)
    c = run(lambda t: t, st)
    for p, q, v in zip(a, b, c):
        assert torch.equal(p, q) and torch.equal(p, v)
    assert np.array_equal(a[0].cpu().numpy(), r.position)


def test_tensor_checks_of_the_python_mirror():
    import torch
    import rccl_amd as ra
    x, out = torch.zeros(4, 64, device="cuda"), torch.zeros(8, 64, device="cuda")
    pos = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    f = ra.ncclFloat32
    for call in (lambda: ra.expert_dispatch(x.half(), out, 8, f, 4, 2, 64, pos),
                 lambda: ra.expert_dispatch(x[:3], out, 8, f, 4, 2, 64, pos),
                 lambda: ra.expert_dispatch(x, out[:, :32], 8, f, 4, 2, 64, pos),
                 lambda: ra.expert_dispatch(x, out.t(), 8, f, 4, 2, 8, pos),
                 lambda: ra.expert_dispatch(x, out, 8, f, 4, 2, 64, pos.long()),
                 lambda: ra.expert_dispatch(x, out, 8, f, 4, 2, 64, pos[:, :1]),
                 lambda: ra.expert_dispatch(x.cpu(), out, 8, f, 4, 2, 64, pos),
                 lambda: ra.expert_dispatch(x, x, 4, f, 4, 2, 64, pos),
                 lambda: ra.expert_dispatch(x, out, 8, f, 4, 2, 64, pos, offsets=torch.zeros(5, dtype=torch.int32, device="cuda"), n_experts=4),
                 lambda: ra.expert_combine(out, 8, torch.zeros(4, 2, device="cuda"), ra.ncclFloat16, x, f, 4, 2, 64, pos),
                 lambda: ra.expert_sort(pos, ra.ncclInt32, 4, 2, 0, 4, 1, pos.float()),
                 lambda: ra.expert_sort(torch.zeros(40000, 1, dtype=torch.int32, device="cuda"), ra.ncclInt32, 40000, 1, 0, 4, 1, torch.zeros(40000, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ra.NcclError) as e:
            call()
        assert e.value.code == ra.ncclInvalidArgument
