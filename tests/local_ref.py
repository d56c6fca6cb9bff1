"""References in 64 bits (and, for the 8-bit states, of every single rounding) for the local operators of a sharded training
step: numpy only, written from the formulas in include/rccl_amd.h."""
import numpy as np

U = 2.0 ** -24                       # a rounding to fp32 is off by at most this part of the value
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}      # the same for each type
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}        # spacing of its subnormal numbers


# ------------------------------------------------------------------ e4m3 with power-of-two block scales
def e4m3_values():
    """Value of each of the 256 codes (OCP e4m3: bias 7, no infinities, 0x7F and 0xFF are NaN)."""
    out = np.empty(256)
    for c in range(256):
        s, e, m = -1.0 if c & 0x80 else 1.0, (c >> 3) & 15, c & 7
        out[c] = s * (np.nan if (c & 0x7F) == 0x7F else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return out


E4M3 = e4m3_values()
GRID = E4M3[:0x7F]                   # the non-negative finite values, in order of their codes


def hash32(seed, step, ordinal, index):
    """The 32 random bits of each element (index: uint64 array)."""
    mask = np.uint64(0xFFFFFFFF)

    def mix(x):
        x = np.asarray(x, dtype=np.uint64) & mask
        x = (x ^ (x >> np.uint64(16))) * np.uint64(0x9E3779B1) & mask
        x = (x ^ (x >> np.uint64(15))) * np.uint64(0xAC564B05) & mask
        return x ^ (x >> np.uint64(16))

    index = np.asarray(index, dtype=np.uint64)
    k = mix((seed & 0xFFFFFFFF) + 0x9E3779B9)
    k = mix(int(k) ^ (seed >> 32))
    k = mix(int(k) + (step & 0xFFFFFFFF))
    k = mix(int(k) + ordinal)
    high = index >> np.uint64(32)
    key = np.where(high > 0, mix(k ^ high), k)
    return mix((index & mask) + key)


def mx_scale(x):
    """The scale exponent (byte) of each block of 32: the smallest power of two with which all finite magnitudes are at most 448."""
    out = np.ones(-(-x.size // 32), dtype=np.int64)
    for b in range(out.size):
        block = np.abs(x[32 * b:32 * b + 32])
        most = float(np.max(block[np.isfinite(block)], initial=0.0))
        while out[b] < 247 and most > 448.0 * 2.0 ** (int(out[b]) - 127):
            out[b] += 1
    return out.astype(np.uint8)


def mx_decode(code, scale):
    factor = np.repeat(2.0 ** (scale.astype(np.float64) - 127), 32)[:code.size]
    factor = np.where(np.repeat(scale, 32)[:code.size] == 0, 0.0, factor)
    return E4M3[code] * factor


def mx_encode(x, rnd16, keep_positive):
    """(codes, scales) of fp32 values.  A value between two neighbours of the grid goes to the upper one where its distance
    from the lower one, in 2^20ths of their distance (cut to a whole number), and the 20 random bits together reach 2^20."""
    scale, fine = mx_scale(x), np.isfinite(x)
    x = np.where(fine, x, np.float32(0))
    y = np.abs(x.astype(np.float64)) / np.repeat(2.0 ** (scale.astype(np.float64) - 127), 32)[:x.size]
    # a value below 2^-6 passes through fp32 in the binade above (its 24 bits reach down to 2^-29)
    y = np.where(y < 2.0 ** -6, (y.astype(np.float32) + np.float32(2.0 ** -6)).astype(np.float64) - 2.0 ** -6, y)
    low = np.clip(np.searchsorted(GRID, y, side="right") - 1, 0, GRID.size - 1)
    gap = np.where(low + 1 < GRID.size, GRID[np.minimum(low + 1, GRID.size - 1)] - GRID[low], 32.0)
    part = np.floor((y - GRID[low]) / gap * 2.0 ** 20)
    code = low + (part + (rnd16.astype(np.int64) << 4 | 8) >= 2 ** 20)
    if keep_positive:
        code = np.where((x > 0) & (code == 0), 1, code)
    return np.where(fine, code | np.where(np.signbit(x), 0x80, 0), 0x7F).astype(np.uint8), scale


# ------------------------------------------------------------------ AdamW
def adamw64(p, g, m, v, *, lr, beta1, beta2, eps, weight_decay, step, coef):
    """Updated (p, m, v) in 64 bits, and bounds on what fp32 arithmetic may make of p, m and v.

    m: each term has a rounded constant, the rounded gradient product and its own product (4 roundings), and the sum one.
    v: its second term has a rounded constant, twice the gradient's two roundings, two products (7), and the sum one.
    sqrt(v): half of v's relative error and one rounding (5); times a rounded constant, plus eps: 8 in all, as eps and the
    root are positive.  The quotient adds one rounding, the step size two, the decayed parameter two, the difference one."""
    p, g, m, v = (np.asarray(x, dtype=np.float64) for x in (p, g, m, v))
    g = g * coef
    m2, v2 = beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g
    big = np.abs(beta1 * m) + np.abs((1 - beta1) * g)
    down = np.sqrt(v2) / np.sqrt(1 - beta2 ** step) + eps
    size = lr / (1 - beta1 ** step)
    p2 = p * (1 - lr * weight_decay) - size * m2 / down
    tiny = 2.0 ** -148                                        # what a product below the normal range may lose
    em, ev = 5.1 * U * big + tiny, 8.1 * U * v2 + tiny
    # where v is subnormal its bound is absolute: the root moves by at most the root of it
    er = np.minimum(ev / np.maximum(np.sqrt(v2), 1e-300), np.sqrt(ev)) / np.sqrt(1 - beta2 ** step)
    ed = er + 4.1 * U * down
    low = np.maximum(down - ed, 1e-300)
    eq = em / low + np.abs(m2) * ed / (down * low) + 1.1 * U * (np.abs(m2) + em) / low
    ep = size * (eq + 2.1 * U * (np.abs(m2) + em) / low) + 2.1 * U * np.abs(p) + 1.1 * U * (np.abs(p2)) + tiny
    return p2, m2, v2, ep, em, ev


# ------------------------------------------------------------------ expert order
def expert_sort(ids, first, n, align):
    """(position, source, offsets, counts) with loops."""
    flat = np.asarray(ids).reshape(-1).astype(np.int64)
    key = flat - first
    keep = (flat >= first) & (flat < first + n)
    counts = np.array([int(np.sum(keep & (key == e))) for e in range(n)], dtype=np.int32)
    offsets = np.zeros(n + 1, dtype=np.int32)
    for e in range(n):
        offsets[e + 1] = offsets[e] + -(-int(counts[e]) // align) * align
    position = np.full(flat.size, -1, dtype=np.int32)
    source = np.full(flat.size + n * (align - 1), -1, dtype=np.int32)
    for e in range(n):
        slots = np.flatnonzero(keep & (key == e))
        rows = offsets[e] + np.arange(slots.size)
        position[slots] = rows
        source[rows] = slots
    return position, source, offsets, counts
