"""The local operators and the collectives together, as a training step of two ranks uses them (one process of its own)."""
import os
import subprocess
import sys

import pytest


@pytest.mark.gpu
def test_training_step_of_two_ranks():
    child = os.path.join(os.path.dirname(os.path.abspath(__file__)), "shard_step_child.py")
    r = subprocess.run([sys.executable, child], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "sharded step ok" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


@pytest.mark.gpu
def test_calls_without_the_mirror_module(monkeypatch):
    """Where the CPython module cannot be loaded, the same calls give the same bits through ctypes."""
    import torch
    import rccl_amd as ra
    from rccl_amd import nccl
    tokens, k, n, h = 100, 4, 8, 264
    rows = ra.expert_rows(tokens, k, n, 16)
    gen = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    ids = torch.randint(0, 2 * n, (tokens, k), generator=gen, device="cuda", dtype=torch.int32)
    x, z, w, dy = rand(tokens, h).bfloat16(), rand(rows, h).bfloat16(), rand(tokens, k), rand(tokens, h).bfloat16()
    p0, g0, m0, v0 = rand(5000), rand(5000).bfloat16(), rand(5000), rand(5000).square()

    def run():
        ints = lambda *s: torch.full(s, -7, dtype=torch.int32, device="cuda")  # noqa: E731
        position, source, offsets, counts = ints(tokens, k), ints(rows), ints(n + 1), ints(n)
        out, y, dz, dw = torch.zeros_like(z), torch.zeros_like(x), torch.zeros_like(z), torch.zeros_like(w)
        total = torch.zeros(1, dtype=torch.float64, device="cuda")
        work = torch.empty(ra.sum_squares_bytes(1), dtype=torch.uint8, device="cuda")
        p, m, v = p0.clone(), m0.clone(), v0.clone()
        ra.expert_sort(ids, ra.ncclInt32, tokens, k, 0, n, 16, position, source, offsets, counts)
        ra.expert_dispatch(x, out, rows, ra.ncclBfloat16, tokens, k, h, position, offsets, counts, n)
        ra.expert_combine(z, rows, w, ra.ncclFloat32, y, ra.ncclBfloat16, tokens, k, h, position)
        ra.expert_combine_backward(dy, z, rows, w, ra.ncclFloat32, dz, dw, ra.ncclBfloat16, tokens, k, h, position, offsets, counts, n)
        ra.sum_squares([g0], None, ra.ncclBfloat16, total, work)
        ra.adamw([ra.adamw_tensor(p, g0, m, v)], ra.ncclFloat32, ra.ncclBfloat16, lr=1e-3, step=3, sum_sq=total, max_norm=1.0)
        torch.cuda.synchronize()
        return position, source, offsets, counts, out, y, dz, dw, total, p, m, v

    plain = run()
    monkeypatch.setitem(sys.modules, "rccl_amd._mirror", None)               # (an import of it fails)
    monkeypatch.delattr(ra, "_mirror", raising=False)
    monkeypatch.setattr(nccl, "_mirror", None)
    with pytest.warns(RuntimeWarning, match="_mirror"):
        other = run()
    for a, b in zip(plain, other):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
