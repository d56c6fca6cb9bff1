"""The local operators of a sharded training step, each in its plain form and as the library's call.

Two sets stand around a reduce-scatter / all-gather pair:

* the optimizer step of a rank's shard: the sum of squares of many gradient tensors, and AdamW over many tensors with
  states in 32 bits or in 8 (MX blocks: 32 elements in e4m3 share one power-of-two scale byte);
* expert parallelism: token slots sorted by expert, rows dispatched to that order and combined back with the router's
  weights, and the gradients of both.

`own` selects what run() computes with: elementary torch operations (False) or the calls of rccl_amd (True).
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i32": torch.int32, "i64": torch.int64}
BLOCK = 32          # elements that share a scale byte in an 8-bit state


def listed():
    return [
        # The slots of one decoding step of a small batch: nothing but latency.
        dict(name="sort decode", op="sort", tokens=32, topk=8, experts=128, first=0, local=128, align=1, ids="i32", padded=0.0),
        # A training batch gathered from eight ranks; this rank holds an eighth of the experts, segments are padded for
        # matrix tiles, three per cent of the tokens are padding with expert -1.
        dict(name="sort gathered", op="sort", tokens=65536, topk=8, experts=128, first=16, local=16, align=128, ids="i64", padded=0.03),
        # Rows of a decoding step, moved to expert order.
        dict(name="dispatch decode", op="dispatch", tokens=16, topk=8, experts=64, first=0, local=64, align=1, hidden=4096, dtype="bf16", padded=0.0),
        # A training micro-batch, all experts on this rank.
        dict(name="dispatch train", op="dispatch", tokens=16384, topk=8, experts=64, first=0, local=64, align=128, hidden=4096, dtype="bf16", padded=0.0),
        # The gradient of a dispatch (no weights): odd sizes, fp32.
        dict(name="combine unweighted odd", op="combine", tokens=501, topk=2, experts=16, first=0, local=16, align=8, hidden=1001, dtype="f32", weights="none", padded=0.05),
        # The same micro-batch back in token order, with the router's weights.
        dict(name="combine train", op="combine", tokens=16384, topk=8, experts=64, first=0, local=64, align=128, hidden=4096, dtype="bf16", weights="f32", padded=0.0),
        # Gradients of a combine: a short batch in fp16 with six slots per token.
        dict(name="combine backward f16", op="combine_backward", tokens=333, topk=6, experts=32, first=0, local=32, align=16, hidden=2048, dtype="f16", weights="f16", padded=0.02),
        # Gradients of a combine after an all-gather of tokens: half of the slots belong to experts of other ranks.
        dict(name="combine backward train", op="combine_backward", tokens=16384, topk=8, experts=64, first=32, local=32, align=128, hidden=4096, dtype="bf16", weights="f32", padded=0.0),
        # The many small tensors of a model's norms, biases and odd projections: clipped by the global norm, fp32 throughout.
        dict(name="adamw ragged f32", op="adamw", tensors=200, largest=60000, state="f32", param="f32", grad="f32", copy="none", clip=True, shift=0),
        # A rank's shard of a 1 GiB bf16 gradient bucket over eight ranks: master weights in fp32, a bf16 copy for the all-gather.
        dict(name="adamw shard f32", op="adamw", tensors=1, largest=67108864, state="f32", param="f32", grad="bf16", copy="bf16", clip=False, shift=0),
        # Ragged tensors with 8-bit states whose views start at odd places of a flat buffer.
        dict(name="adamw ragged mx8", op="adamw", tensors=96, largest=90000, state="mx8", param="bf16", grad="bf16", copy="none", clip=False, shift=3),
        # The same shard with 8-bit states, clipped by the global norm.
        dict(name="adamw shard mx8", op="adamw", tensors=1, largest=67108864, state="mx8", param="f32", grad="bf16", copy="bf16", clip=True, shift=0),
    ]


def _spread(rng, lo, hi):
    """A whole number in lo..hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["sort", "dispatch", "combine", "combine_backward", "adamw", "adamw"])
    if op == "adamw":
        n = _spread(rng, 1, 300)
        return dict(op=op, tensors=n, largest=_spread(rng, 1, 67108864 // n), state=rng.choice(["f32", "mx8"]), param=rng.choice(["f32", "f32", "bf16", "f16"]),
                    grad=rng.choice(["f32", "bf16", "f16"]), copy=rng.choice(["none", "bf16", "f16", "f32"]), clip=rng.random() < 0.5, shift=rng.choice([0, 0, 1, 3, 4]))
    experts = _spread(rng, 1, 384)
    topk = rng.randint(1, min(10, experts))
    part = rng.choice([1, 1, 2, 4, 8])
    local = max(1, experts // part)
    first = rng.randrange(0, experts - local + 1)
    c = dict(op=op, topk=topk, experts=experts, first=first, local=local, align=rng.choice([1, 1, 8, 16, 100, 128]), padded=rng.choice([0.0, 0.0, 0.03, 0.5]))
    if op == "sort":
        return dict(c, tokens=_spread(rng, 1, 524288 // topk), ids=rng.choice(["i32", "i64"]))
    c["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
    c["hidden"] = _spread(rng, 1, 8192)
    most = min(65536, 16384 * 8 * 4096 // (topk * c["hidden"] * (2 if c["dtype"] == "f32" else 1)))
    c["tokens"] = _spread(rng, 1, max(1, most))
    if op != "dispatch":
        c["weights"] = rng.choice(["f32", "f32", "bf16", "f16"]) if op == "combine_backward" else rng.choice(["none", "f32", "bf16", "f16"])
    return c


# ---------------------------------------------------------------------------------------------- what each case has to move
def _size(name):
    return 0 if name == "none" else torch.empty(0, dtype=TYPES[name]).element_size()


def _sizes(case):
    """The element counts of an AdamW case's tensors: one of the largest size, the others spread below it."""
    rng = np.random.RandomState(case["tensors"] * 7919 + case["largest"] % 104729)
    small = np.exp(rng.uniform(0, math.log(case["largest"] + 0.49), case["tensors"] - 1)).astype(np.int64)
    return np.concatenate([np.array([case["largest"]], dtype=np.int64), np.clip(small, 1, case["largest"])])


def _rows(case):
    """Rows of the sorted order: its slots, and up to align - 1 rows of padding for each expert."""
    return case["tokens"] * case["topk"] + case["local"] * (case["align"] - 1)


def work(case):
    if case["op"] == "adamw":
        n = float(_sizes(case).sum())
        state = 2 * (8.0 if case["state"] == "f32" else 2 + 2.0 / BLOCK)
        each = 2 * _size(case["param"]) + _size(case["grad"]) + _size(case["copy"]) + state
        return {"bytes": n * each, "flops": n * (16 + (2 if case["clip"] else 0))}
    slots = case["tokens"] * case["topk"]
    held = slots * (1 - case["padded"]) * case["local"] / case["experts"]      # slots of this rank's experts, as routing goes
    rows = held + case["local"] * (case["align"] - 1) / 2.0
    if case["op"] == "sort":
        return {"bytes": slots * (_size(case["ids"]) + 4.0) + 4.0 * _rows(case) + 8.0 * case["local"] + 4, "flops": float(slots)}
    touched = case["tokens"] * (1 - case["padded"]) * (1 - (1 - case["local"] / case["experts"]) ** case["topk"])   # tokens with a slot here
    row = float(case["hidden"] * _size(case["dtype"]))
    if case["op"] == "dispatch":
        return {"bytes": touched * row + rows * row + 4.0 * slots, "flops": rows * case["hidden"]}
    w = slots * (4.0 + _size(case["weights"]))
    if case["op"] == "combine":
        return {"bytes": held * row + case["tokens"] * row + w, "flops": 2.0 * held * case["hidden"]}
    return {"bytes": touched * row + held * row + rows * row + w + slots * _size(case["weights"]), "flops": 3.0 * held * case["hidden"]}


# ---------------------------------------------------------------------------------------------- inputs
def _routing(case, gen):
    """Expert ids of a router with favourites: the top k of random scores with a bias for each expert; padding tokens have -1."""
    t, e = case["tokens"], case["experts"]
    score = torch.randn(t, e, generator=gen, device="cuda") + 0.7 * torch.randn(e, generator=gen, device="cuda")
    ids = score.topk(case["topk"], dim=1).indices
    live = torch.rand(t, 1, generator=gen, device="cuda") >= case["padded"]
    return torch.where(live, ids, -1)


def _sort(ids, case):
    """(position, source, offsets, counts) by elementary operations: see run()."""
    n, a, rows = case["local"], case["align"], _rows(case)
    key = ids.reshape(-1).to(torch.int64) - case["first"]
    key = torch.where((key >= 0) & (key < n), key, n)
    key, order = torch.sort(key, stable=True)
    start = torch.searchsorted(key, torch.arange(n + 1, device=key.device))
    counts = start[1:] - start[:-1]
    offsets = torch.zeros(n + 1, dtype=torch.int64, device=key.device)
    offsets[1:] = torch.cumsum((counts + (a - 1)) // a * a, 0)
    place = offsets[key] + torch.arange(key.numel(), device=key.device) - start[key]
    place = torch.where(key < n, place, rows)                      # row `rows` takes what is dropped
    source = torch.full((rows + 1,), -1, dtype=torch.int32, device=key.device)
    source[place] = order.to(torch.int32)
    position = torch.empty(key.numel(), dtype=torch.int32, device=key.device)
    position[order] = torch.where(key < n, place, -1).to(torch.int32)
    return position.view(case["tokens"], case["topk"]), source[:rows], offsets.to(torch.int32), counts.to(torch.int32)


def _blocks(x):
    return x.view(-1, BLOCK)


def _encode(value, rnd, live, keep_positive):
    """MX encoding of a flat run of blocks: (e4m3 elements, scale bytes).  The scale is the smallest power of two with which
    the block's largest magnitude is at most 448; `rnd`, 20 random bits for each value, goes below the mantissa's third bit
    (below 2^-9 in the subnormal range) before the rest is cut off.  `keep_positive`: a value over zero is not rounded to it."""
    bits = torch.where(live, value.view(torch.int32) & 0x7FFFFFFF, 0)
    most = _blocks(bits).amax(1, keepdim=True).to(torch.int64)
    e = (((most + 0x1FFFFF) >> 23) - 8).clamp(1, 247)
    inverse = ((254 - e) << 23).to(torch.int32).view(torch.float32)
    y = (_blocks(value) * inverse).view(-1)
    a = y.abs()
    low = torch.where(a < 2.0 ** -6, 2.0 ** -6, 0.0).to(torch.float32)
    cut = ((a + low).view(torch.int32) + rnd) & ~0xFFFFF
    a2 = cut.view(torch.float32) - low
    if keep_positive:
        a2 = torch.where(value > 0, torch.clamp(a2, min=2.0 ** -9), a2)
    y2 = torch.where(torch.isfinite(y), torch.copysign(a2, y), float("nan"))
    return y2.to(torch.float8_e4m3fn), e.to(torch.uint8).view(-1)


def _decode(code, scale):
    factor = (scale.to(torch.int32) << 23).view(torch.float32)
    return (_blocks(code.to(torch.float32)) * factor[:, None]).view(-1)


def _shifted(n, dtype, shift, fill=None):
    """A flat run of n elements that starts `shift` elements into its storage."""
    t = torch.zeros(n + shift + 8, dtype=dtype, device="cuda")[shift:shift + n]
    if fill is not None:
        t.copy_(fill)
    return t


def _prepare_adamw(case, gen):
    sizes = _sizes(case)
    begin = np.concatenate([[0], np.cumsum((sizes + BLOCK - 1) // BLOCK * BLOCK)])   # every tensor starts at a block
    n = int(begin[-1])
    host = np.repeat(np.arange(len(sizes)), np.diff(begin))
    ordinal = torch.from_numpy(host).cuda()
    index = torch.arange(n, device="cuda") - torch.from_numpy(begin[:-1]).cuda()[ordinal]
    live = index < torch.from_numpy(sizes).cuda()[ordinal]
    loud = torch.exp(torch.randn(len(sizes), generator=gen, device="cuda"))[ordinal]      # each tensor has a gradient scale of its own
    rand = lambda: torch.randn(n, generator=gen, device="cuda")  # noqa: E731
    s = dict(case=case, n=n, live=live, ordinal=ordinal.to(torch.int32), index=index.to(torch.int32), blocks=n // BLOCK)
    sh = case["shift"]
    s["param"] = _shifted(n, TYPES[case["param"]], sh, 0.02 * rand())
    s["grad"] = _shifted(n, TYPES[case["grad"]], sh, 1e-3 * loud * rand())
    s["copy"] = None if case["copy"] == "none" else _shifted(n, TYPES[case["copy"]], sh)
    m, v = 3e-4 * loud * rand(), (1e-3 * loud * rand().abs().add_(0.05)).square_()
    if case["state"] == "f32":
        s["m"], s["v"] = _shifted(n, torch.float32, sh, m), _shifted(n, torch.float32, sh, v)
        s["ms"] = s["vs"] = None
    else:
        half = torch.full((n,), 1 << 19, dtype=torch.int32, device="cuda")
        s["m"], s["ms"] = _encode(m, half, live, False)
        s["v"], s["vs"] = _encode(v.sqrt(), half, live, True)
        s["m"], s["v"] = (_shifted(n, torch.uint8, sh, x.view(torch.uint8)) for x in (s["m"], s["v"]))
    del m, v, loud
    s.update(lr=3e-4, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1, step=1000, grad_scale=0.5, max_norm=1.0,
             seed=int(torch.randint(0, 2 ** 62, (1,), generator=gen, device="cuda").item()))
    s["sum_sq"] = torch.zeros(1, dtype=torch.float64, device="cuda")
    # The table a program keeps: a row for each tensor with the addresses of its parameter, gradient, both moments, their
    # scales and its copy, and its size (0 where there is none).
    table = np.zeros((len(sizes), 8), dtype=np.int64)
    for col, key in enumerate(("param", "grad", "m", "v", "ms", "vs", "copy")):
        if s[key] is not None:
            first = begin[:-1] // BLOCK if key in ("ms", "vs") else begin[:-1]
            table[:, col] = s[key].data_ptr() + first * s[key].element_size()
    table[:, 7] = sizes
    s["table"], s["grads"], s["sizes"] = table, np.ascontiguousarray(table[:, 1]), sizes
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "adamw":
        return _prepare_adamw(case, gen)
    ids = _routing(case, gen)
    rows, slots = _rows(case), case["tokens"] * case["topk"]
    if case["op"] == "sort":
        return dict(case=case, ids=ids.to(TYPES[case["ids"]]), position=torch.empty(case["tokens"], case["topk"], dtype=torch.int32, device="cuda"),
                    source=torch.empty(rows, dtype=torch.int32, device="cuda"), offsets=torch.empty(case["local"] + 1, dtype=torch.int32, device="cuda"),
                    counts=torch.empty(case["local"], dtype=torch.int32, device="cuda"))
    dt, h = TYPES[case["dtype"]], case["hidden"]
    s = dict(case=case)
    s["position"], s["source"], s["offsets"], s["counts"] = _sort(ids, case)
    s["position"] = s["position"].contiguous()
    fill = lambda r: torch.randn(r, h, generator=gen, device="cuda").to(dt)  # noqa: E731
    if case["op"] in ("combine", "combine_backward"):
        s["z"] = fill(rows)
        s["weights"] = None
        if case["weights"] != "none":
            s["weights"] = torch.softmax(torch.randn(case["tokens"], case["topk"], generator=gen, device="cuda"), 1).to(TYPES[case["weights"]])
    if case["op"] == "dispatch":
        s["x"] = fill(case["tokens"])
        s["out"] = torch.zeros(rows, h, dtype=dt, device="cuda")
    elif case["op"] == "combine":
        s["y"] = torch.empty(case["tokens"], h, dtype=dt, device="cuda")
    else:
        s["dy"] = fill(case["tokens"])
        s["dz"] = torch.zeros(rows, h, dtype=dt, device="cuda")
        s["dw"] = torch.empty(case["tokens"], case["topk"], dtype=TYPES[case["weights"]], device="cuda")
    return s


# ---------------------------------------------------------------------------------------------- the plain forms
def _mix(x):
    x = (x ^ (x >> 16)) * 0x9E3779B1 & 0xFFFFFFFF
    x = (x ^ (x >> 15)) * 0xAC564B05 & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random(s):
    """32 random bits for each element: a hash of the seed, the step, the tensor's place in the table and the element's in the tensor."""
    k = _mix((s["seed"] & 0xFFFFFFFF) + 0x9E3779B9 & 0xFFFFFFFF)
    k = _mix(k ^ (s["seed"] >> 32))
    k = _mix(k + s["step"] & 0xFFFFFFFF)
    k = _mix((s["ordinal"].to(torch.int64) + k) & 0xFFFFFFFF)
    return _mix((s["index"].to(torch.int64) + k) & 0xFFFFFFFF)


def _adamw(s):
    case, live = s["case"], s["live"]
    g = s["grad"].to(torch.float32)
    old = s["param"].to(torch.float32)
    fine = live
    if case["clip"]:
        square = torch.where(live, s["grad"], 0).to(torch.float64).square().sum()
        s["sum_sq"].copy_(square.view(1))
        c = s["grad_scale"] * torch.clamp(s["max_norm"] / (s["grad_scale"] * square.sqrt() + 1e-6), max=1.0)
        g = g * c.to(torch.float32)
        fine = live & torch.isfinite(square)          # a norm that is not finite leaves all as it was
    else:
        g = g * s["grad_scale"]
    m0, v0 = s["m"], s["v"]
    if case["state"] == "mx8":
        m0, r0 = _decode(m0.view(torch.float8_e4m3fn), s["ms"]), _decode(v0.view(torch.float8_e4m3fn), s["vs"])
        v0 = r0 * r0
    m = s["beta1"] * m0 + (1 - s["beta1"]) * g
    v = s["beta2"] * v0 + (1 - s["beta2"]) * (g * g)
    r = torch.sqrt(v)
    down = r * (1 / math.sqrt(1 - s["beta2"] ** s["step"])) + s["eps"]
    p = old * (1 - s["lr"] * s["weight_decay"]) - (s["lr"] / (1 - s["beta1"] ** s["step"])) * (m / down)
    s["param"].copy_(torch.where(fine, p, old))
    if s["copy"] is not None:
        s["copy"].copy_(torch.where(live, torch.where(fine, p, old), s["copy"].to(torch.float32)))
    if case["state"] == "f32":
        s["m"].copy_(torch.where(fine, m, s["m"]))
        s["v"].copy_(torch.where(fine, v, s["v"]))
    else:
        h = _random(s)
        go = _blocks(fine).any(1)
        for key, scale, x, rnd, up in (("m", "ms", m, h & 0xFFFF, False), ("v", "vs", r, h >> 16, True)):
            code, e = _encode(x, (rnd << 4 | 8).to(torch.int32), live, up)
            s[key].copy_(torch.where(fine, code.view(torch.uint8), s[key]))
            s[scale].copy_(torch.where(go, e, s[scale]))


def _gathered(rows, position):
    """rows[position] in fp32 for each slot, zeros where the slot is dropped."""
    return torch.where((position >= 0)[..., None], rows[position.clamp(min=0).to(torch.int64)].to(torch.float32), 0.0)


def _plain(s):
    case = s["case"]
    if case["op"] == "adamw":
        _adamw(s)
    elif case["op"] == "sort":
        s["position"], s["source"], s["offsets"], s["counts"] = _sort(s["ids"], case)
    elif case["op"] == "combine":
        z = _gathered(s["z"], s["position"])
        if s["weights"] is not None:
            z = z * s["weights"].to(torch.float32)[..., None]
        s["y"] = z.sum(1).to(s["z"].dtype)
    else:
        source, rows = s["source"].to(torch.int64), _rows(case)
        token = source.clamp(min=0) // case["topk"]
        inside = torch.arange(rows, device="cuda") < s["offsets"][-1]
        if case["op"] == "dispatch":
            moved = torch.where((source >= 0)[:, None], s["x"][token], 0)
            s["out"].copy_(torch.where(inside[:, None], moved, s["out"]))
        else:
            w = s["weights"].to(torch.float32).reshape(-1)[source.clamp(min=0)]
            moved = torch.where((source >= 0)[:, None], s["dy"][token].to(torch.float32) * w[:, None], 0.0)
            s["dz"].copy_(torch.where(inside[:, None], moved, s["dz"].to(torch.float32)))
            s["dw"] = (_gathered(s["z"], s["position"]) * s["dy"].to(torch.float32)[:, None, :]).sum(2).to(s["weights"].dtype)


# ---------------------------------------------------------------------------------------------- the library's calls
def _workspace(s, nbytes):
    if "workspace" not in s:
        s["workspace"] = torch.empty(max(1, nbytes), dtype=torch.uint8, device="cuda")
    return s["workspace"]


def _library(s):
    import rccl_amd as ra
    case = s["case"]
    kind = {"f32": ra.ncclFloat32, "bf16": ra.ncclBfloat16, "f16": ra.ncclFloat16, "i32": ra.ncclInt32, "i64": ra.ncclInt64, "none": -1}
    if case["op"] == "adamw":
        if case["clip"]:
            ra.sum_squares(s["grads"], s["sizes"], kind[case["grad"]], s["sum_sq"], _workspace(s, ra.sum_squares_bytes(len(s["sizes"]))))
        ra.adamw(s["table"], kind[case["param"]], kind[case["grad"]], kind[case["copy"]], ra.rcclAmdStateF32 if case["state"] == "f32" else ra.rcclAmdStateMx8,
                 lr=s["lr"], beta1=s["beta1"], beta2=s["beta2"], eps=s["eps"], weight_decay=s["weight_decay"], step=s["step"], grad_scale=s["grad_scale"],
                 sum_sq=s["sum_sq"] if case["clip"] else None, max_norm=s["max_norm"], seed=s["seed"])
    elif case["op"] == "sort":
        ra.expert_sort(s["ids"], kind[case["ids"]], case["tokens"], case["topk"], case["first"], case["local"], case["align"], s["position"], s["source"],
                       s["offsets"], s["counts"], _workspace(s, ra.expert_sort_bytes(case["tokens"], case["topk"], case["local"])))
    elif case["op"] == "dispatch":
        ra.expert_dispatch(s["x"], s["out"], _rows(case), kind[case["dtype"]], case["tokens"], case["topk"], case["hidden"], s["position"],
                           offsets=s["offsets"], counts=s["counts"], n_experts=case["local"])
    elif case["op"] == "combine":
        ra.expert_combine(s["z"], _rows(case), s["weights"], kind[case["weights"]], s["y"], kind[case["dtype"]], case["tokens"], case["topk"], case["hidden"], s["position"])
    else:
        ra.expert_combine_backward(s["dy"], s["z"], _rows(case), s["weights"], kind[case["weights"]], s["dz"], s["dw"], kind[case["dtype"]], case["tokens"], case["topk"],
                                   case["hidden"], s["position"], offsets=s["offsets"], counts=s["counts"], n_experts=case["local"])


def run(state):
    if own:
        _library(state)
    else:
        _plain(state)
    op = state["case"]["op"]
    if op == "adamw":
        out = {"param": state["param"], "sum_sq": state["sum_sq"]}
        if state["copy"] is not None:
            out["copy"] = state["copy"]
        if state["case"]["state"] == "f32":
            return dict(out, m=state["m"], v=state["v"])
        return dict(out, m=state["m"].view(torch.float8_e4m3fn), root_v=state["v"].view(torch.float8_e4m3fn), m_scale=state["ms"], root_v_scale=state["vs"])
    if op == "sort":
        return {k: state[k] for k in ("position", "source", "offsets", "counts")}
    return {"dispatch": lambda: state["out"], "combine": lambda: state["y"], "combine_backward": lambda: {"dz": state["dz"], "dw": state["dw"]}}[op]()


# ---------------------------------------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sort":
        return None                                     # whole numbers only
    if case["op"] == "adamw":
        f = lambda x: x.to(torch.float64)  # noqa: E731
        live = s["live"]
        total = (f(s["grad"]) * live).pow(2).sum()
        g = f(s["grad"]) * s["grad_scale"]
        if case["clip"]:
            g = g * min(1.0, s["max_norm"] / (s["grad_scale"] * math.sqrt(float(total)) + 1e-6))
        if case["state"] == "f32":
            m, v = f(s["m"]), f(s["v"])
        else:
            each = lambda key, scale: f(s[key].view(torch.float8_e4m3fn).to(torch.float32)) * torch.exp2(f(s[scale]) - 127).repeat_interleave(BLOCK)  # noqa: E731
            m, v = each("m", "ms"), each("v", "vs").pow(2)
        m = torch.where(live, m + (1 - s["beta1"]) * (g - m), m)
        v = torch.where(live, v + (1 - s["beta2"]) * (g * g - v), v)
        hat_m, hat_v = m / (1 - s["beta1"] ** s["step"]), v / (1 - s["beta2"] ** s["step"])
        old = f(s["param"])
        p = torch.where(live, old - s["lr"] * (hat_m / (hat_v.sqrt() + s["eps"]) + s["weight_decay"] * old), old)
        out = {"param": p, "sum_sq": total.view(1) if case["clip"] else f(s["sum_sq"])}
        if s["copy"] is not None:
            out["copy"] = torch.where(live, p, 0.0)
        if case["state"] == "f32":
            return dict(out, m=m, v=v)
        # An element that is rounded to 8 bits by a random number has no value in 64 bits.
        return dict(out, m=None, root_v=None, m_scale=None, root_v_scale=None)
    position, k = s["position"].to(torch.int64), case["topk"]
    weights = s["weights"].to(torch.float64) if s.get("weights") is not None else None
    if case["op"] == "combine":
        y = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
        for j in range(k):
            has = position[:, j] >= 0
            part = s["z"][position[has, j]].to(torch.float64)
            y[has] += part if weights is None else part * weights[has, j, None]
        return y
    rows = s["x"] if case["op"] == "dispatch" else s["dy"]
    moved = torch.zeros(_rows(case), case["hidden"], dtype=torch.float64, device="cuda")
    dw = torch.zeros(case["tokens"], k, dtype=torch.float64, device="cuda")
    for j in range(k):
        has = position[:, j] >= 0
        part = rows[has].to(torch.float64)
        if case["op"] == "combine_backward":
            dw[has, j] = (part * s["z"][position[has, j]].to(torch.float64)).sum(1)
            part = part * weights[has, j, None]
        moved[position[has, j]] = part
    return moved if case["op"] == "dispatch" else {"dz": moved, "dw": dw}
