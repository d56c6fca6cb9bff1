"""A training step of two ranks (both on GPU 0, one process) through the collectives and the local operators together:
a layer of experts, half of them on each rank, over all-gather and reduce-scatter, forward and backward, and then the clipped
AdamW step of a sharded parameter between reduce-scatter and all-gather.  Checked against numpy in 64 bits.  Run by
tests/test_gpu_kernels_step.py in a process of its own: the communicators' windows live until it ends."""
import math
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "tests")]
os.environ["RCCL_AMD_MULTI_RANK_GPU"] = "1"
os.environ.setdefault("RCCL_AMD_SPIN_TIMEOUT_MS", "10000")

import numpy as np  # noqa: E402
import torch  # noqa: E402

import local_ref as ref  # noqa: E402
import rccl_amd as ra  # noqa: E402

N, T, K, H, E = 2, 96, 2, 64, 8                # ranks, tokens of each, slots, elements, experts
LOCAL, ALIGN = E // N, 8
F = ra.ncclFloat32


def main():
    torch.cuda.set_device(0)
    comms = ra.Communicator.init_all(N, [0] * N)
    streams = [torch.cuda.Stream() for _ in range(N)]
    rng = np.random.default_rng(0)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    zeros = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731

    def together(call):
        """call(rank) for both ranks as one group, finished before anything else runs."""
        torch.cuda.synchronize()
        ra.group_start()
        for r in range(N):
            call(r)
        ra.group_end()
        torch.cuda.synchronize()
        for c in comms:
            assert c.async_error() == 0

    def gathered(parts, kind):
        outs = [zeros(N * parts[0].shape[0], *parts[0].shape[1:], dtype=parts[0].dtype) for _ in range(N)]
        together(lambda r: comms[r].all_gather(parts[r], outs[r], parts[r].numel(), kind, streams[r]))
        return outs

    def scattered(wholes, kind):
        outs = [zeros(w.shape[0] // N, *w.shape[1:], dtype=w.dtype) for w in wholes]
        together(lambda r: comms[r].reduce_scatter(wholes[r], outs[r], outs[r].numel(), kind, ra.ncclSum, streams[r]))
        return outs

    # ---- a layer of experts -----------------------------------------------------------------------------------------
    x = rng.standard_normal((N * T, H)).astype(np.float32)
    ids = np.argsort(rng.random((N * T, E)), axis=1)[:, :K].astype(np.int32)
    ids[rng.random(N * T) < 0.1] = -1
    w = rng.random((N * T, K)).astype(np.float32)
    dy = rng.standard_normal((N * T, H)).astype(np.float32)
    mats = (rng.standard_normal((E, H, H)) / 8).astype(np.float32)
    mine = lambda a, r: dev(a[r * T:(r + 1) * T])  # noqa: E731
    xs, idss, ws = gathered([mine(x, r) for r in range(N)], F), gathered([mine(ids, r) for r in range(N)], ra.ncclInt32), gathered([mine(w, r) for r in range(N)], F)
    rows = ra.expert_rows(N * T, K, LOCAL, ALIGN)
    partial, kept = [], []
    for r in range(N):
        s = dict(position=zeros(N * T, K, dtype=torch.int32), offsets=zeros(LOCAL + 1, dtype=torch.int32), counts=zeros(LOCAL, dtype=torch.int32), out=zeros(rows, H), z=zeros(rows, H))
        ra.expert_sort(idss[r], ra.ncclInt32, N * T, K, r * LOCAL, LOCAL, ALIGN, s["position"], None, s["offsets"], s["counts"])
        seg = dict(offsets=s["offsets"], counts=s["counts"], n_experts=LOCAL)
        ra.expert_dispatch(xs[r], s["out"], rows, F, N * T, K, H, s["position"], **seg)
        off = s["offsets"].tolist()
        for e in range(LOCAL):
            s["z"][off[e]:off[e + 1]] = s["out"][off[e]:off[e + 1]] @ dev(mats[r * LOCAL + e])
        y = zeros(N * T, H)
        ra.expert_combine(s["z"], rows, ws[r], F, y, F, N * T, K, H, s["position"])
        partial.append(y)
        kept.append((s, seg, off))
    y = torch.cat(scattered(partial, F)).double().cpu().numpy()
    dys = gathered([mine(dy, r) for r in range(N)], F)
    dxs, dws, dmats = [], [], np.zeros((E, H, H))
    for r in range(N):
        s, seg, off = kept[r]
        dz, dw, dout, dx = zeros(rows, H), zeros(N * T, K), zeros(rows, H), zeros(N * T, H)
        ra.expert_combine_backward(dys[r], s["z"], rows, ws[r], F, dz, dw, F, N * T, K, H, s["position"], **seg)
        for e in range(LOCAL):
            cut = slice(off[e], off[e + 1])
            dmats[r * LOCAL + e] = (s["out"][cut].T @ dz[cut]).double().cpu().numpy()
            dout[cut] = dz[cut] @ dev(mats[r * LOCAL + e]).T
        ra.expert_combine(dout, rows, None, -1, dx, F, N * T, K, H, s["position"])
        dxs.append(dx), dws.append(dw)
    dx, dw = torch.cat(scattered(dxs, F)).double().cpu().numpy(), torch.cat(scattered(dws, F)).double().cpu().numpy()

    a, b, m64 = x.astype(np.float64), dy.astype(np.float64), mats.astype(np.float64)
    want = {n: np.zeros(sh) for n, sh in (("y", a.shape), ("dx", a.shape), ("dw", (N * T, K)), ("dmats", m64.shape))}
    size = {n: np.zeros_like(v) for n, v in want.items()}                # sums of the magnitudes of the same terms
    for t in range(N * T):
        for k in range(K):
            e = ids[t, k]
            if e >= 0:
                for into, f in ((want, lambda v: v), (size, np.abs)):
                    z = f(a[t]) @ f(m64[e])
                    into["y"][t] += w[t, k] * z
                    into["dw"][t, k] = f(b[t]) @ z
                    into["dx"][t] += w[t, k] * (f(m64[e]) @ f(b[t]))
                    into["dmats"][e] += w[t, k] * np.outer(f(a[t]), f(b[t]))
    # every result is a sum of products in fp32: at most 64 + 64 + 10 roundings on the way to it, or, for the experts'
    # gradients, as many as there are tokens and a few
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("dmats", dmats)):
        assert np.all(np.abs(got - want[name]) <= (N * T + 10) * ref.U * size[name]), name
    print("layer ok", flush=True)

    # ---- the optimizer step of a sharded parameter ------------------------------------------------------------------
    count = 10_000                              # elements of each shard: three tensors that end inside it
    cuts = [0, 1000, 1001, count]
    grads = (1e-2 * rng.standard_normal((N, N * count))).astype(np.float32)
    bf = lambda a: torch.from_numpy(a).to(torch.bfloat16)  # noqa: E731
    shards = scattered([bf(grads[r]).cuda() for r in range(N)], ra.ncclBfloat16)
    master = [dev(rng.standard_normal(count).astype(np.float32)) for _ in range(N)]
    before = [p.double().cpu().numpy() for p in master]
    model = [zeros(N * count, dtype=torch.bfloat16) for _ in range(N)]             # the all-gather is in place
    states = [[zeros(count), zeros(count)] for _ in range(N)]
    sums = [zeros(1, dtype=torch.float64) for _ in range(N)]
    work = zeros(ra.sum_squares_bytes(3), dtype=torch.uint8)
    for r in range(N):
        ra.sum_squares([shards[r][i:j] for i, j in zip(cuts, cuts[1:])], None, ra.ncclBfloat16, sums[r], work)
    together(lambda r: comms[r].all_reduce(sums[r], sums[r], 1, ra.ncclFloat64, ra.ncclSum, streams[r]))
    norm = math.sqrt(sum(float((s.double() ** 2).sum()) for s in shards))
    assert all(abs(float(s) / norm ** 2 - 1) < 1e-12 for s in sums) and float(sums[0]) == float(sums[1])
    hyper = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1, step=1)
    for r in range(N):
        copy = model[r][r * count:(r + 1) * count]
        table = [ra.adamw_tensor(master[r][i:j], shards[r][i:j], states[r][0][i:j], states[r][1][i:j], copy=copy[i:j]) for i, j in zip(cuts, cuts[1:])]
        ra.adamw(table, F, ra.ncclBfloat16, ra.ncclBfloat16, sum_sq=sums[r], max_norm=0.5 * norm, grad_scale=0.5, **hyper)
    together(lambda r: comms[r].all_gather(model[r][r * count:(r + 1) * count], model[r], count, ra.ncclBfloat16, streams[r]))
    assert torch.equal(model[0], model[1])
    coef = 0.5 * min(1.0, 0.5 * norm / (0.5 * norm + 1e-6))
    for r in range(N):
        want, _, _, bound, _, _ = ref.adamw64(before[r], shards[r].double().cpu().numpy(), 0, 0, coef=coef, **hyper)
        assert np.all(np.abs(master[r].double().cpu().numpy() - want) <= bound)
        assert torch.equal(model[1 - r][r * count:(r + 1) * count], master[r].to(torch.bfloat16))
    for c in comms:
        c.destroy()
    print("sharded step ok", flush=True)


if __name__ == "__main__":
    main()
