"""Argument checks and host logic of the local operators (no GPU: every call here is refused before anything is launched,
or has nothing to do)."""
import ctypes
import os
import subprocess
import sys
import sysconfig

import numpy as np
import pytest

import rccl_amd as ra

P = 0x10000                      # a device pointer that is never followed: the calls below are refused


def _refused(call, text):
    with pytest.raises(ra.NcclError) as e:
        call()
    assert e.value.code == ra.ncclInvalidArgument and text in str(e.value), str(e.value)


def _adamw(rows=None, **kw):
    rows = [[P, P, P, P, P, P, 0, 100]] if rows is None else rows
    args = dict(param_type=ra.ncclFloat32, grad_type=ra.ncclFloat32, copy_type=-1, state_type=ra.rcclAmdStateF32, lr=1e-3, step=1, stream=0)
    args.update(kw)
    ra.adamw(np.array(rows, dtype=np.int64), **args)


@pytest.mark.parametrize("kw,text", [
    (dict(param_type=ra.ncclFloat64), "parameter type"), (dict(grad_type=ra.ncclInt32), "gradient type"), (dict(state_type=2), "state type"),
    (dict(lr=float("nan")), "finite"), (dict(eps=-1.0), "eps"), (dict(weight_decay=float("inf")), "finite"), (dict(grad_scale=float("nan")), "finite"), (dict(grad_scale=-1.0), "negative"),
    (dict(beta1=1.0), "beta1"), (dict(beta2=-0.1), "beta"), (dict(beta2=float("nan")), "beta"), (dict(step=0), "first step"),
    (dict(sum_sq=P, max_norm=-1.0), "maxNorm"), (dict(sum_sq=P, max_norm=float("nan")), "maxNorm"), (dict(sum_sq=P + 4), "misaligned"), (dict(step_ptr=P + 2), "misaligned"),
    (dict(rows=[[0, P, P, P, 0, 0, 0, 1]]), "null buffer"), (dict(rows=[[P, P, P, 0, 0, 0, 0, 1]]), "null buffer"),
    (dict(rows=[[P, P, P, P, 0, P, 0, 1]], state_type=1), "null buffer"),
    (dict(rows=[[P + 2, P, P, P, 0, 0, 0, 1]]), "aligned"), (dict(rows=[[P, P + 1, P, P, 0, 0, 0, 1]], grad_type=ra.ncclBfloat16), "aligned"),
    (dict(rows=[[P, P, P + 1, P, 0, 0, 0, 1]]), "aligned"), (dict(rows=[[P, P, P, P, 0, 0, P + 1, 1]], copy_type=ra.ncclBfloat16), "aligned"),
    (dict(rows=[[P, P, P, P, 0, 0, P, 1]]), "copy type"), (dict(rows=[[P, P, P, P, 0, 0, 0, 2 ** 62]]), "elements"),
    (dict(rows=[[P, P, P, P, 0, 0, 0, 2 ** 42]] * 3), "elements"),
])
def test_adamw_refusals(kw, text):
    _refused(lambda: _adamw(**kw), text)


@pytest.mark.parametrize("eps", [1e-40, 2.0 ** -127, 5e-324])
def test_adamw_refuses_an_eps_that_fp32_does_not_hold_as_a_normal_number(eps):
    _refused(lambda: _adamw(eps=eps), "normal fp32")


@pytest.mark.parametrize("eps", [2.0 ** 128, 1e39, 1.7e308])
@pytest.mark.parametrize("state_type", [0, 1])
def test_adamw_refuses_an_eps_that_is_infinite_in_fp32(eps, state_type):
    _refused(lambda: _adamw(eps=eps, state_type=state_type, rows=[[P, P, P, P, P * state_type, P * state_type, 0, 100]]), "normal fp32")


@pytest.mark.parametrize("eps", [2.0 ** 127, 3e38, float(np.nextafter(2.0 ** 126, np.inf))])
def test_adamw_refuses_an_eps_without_a_normal_reciprocal_for_8_bit_states(eps):
    _refused(lambda: _adamw(eps=eps, state_type=1), "2^126")
    _refused(lambda: _adamw(eps=eps, rows=[[0, P, P, P, 0, 0, 0, 1]]), "null buffer")      # 32-bit states: eps is taken, the row is not


@pytest.mark.parametrize("scales", [(P, P), (P, 0), (0, P)])
@pytest.mark.parametrize("ntensors", [1, 200])
def test_adamw_refuses_8_bit_moments_as_floats(scales, ntensors):
    """A row with scales names moments of one byte each; with 32-bit states they would be read and written past their end."""
    rows = [[P, P, P, P, *(scales if i == ntensors - 1 else (0, 0)), 0, 100] for i in range(ntensors)]
    _refused(lambda: _adamw(rows=rows), "has scales")


def test_adamw_without_work():
    _adamw(rows=np.zeros((0, 8)))
    _adamw(rows=[[0] * 8] * 200)                               # empty tensors need no buffers
    L = ra.lib()
    assert L.rcclAmdAdamW(None, 0, 7, 7, 7, 0, None, None) == ra.ncclInvalidArgument      # a configuration is always needed
    c = ra.rcclAmdAdamWConfig_t(step=1)
    assert L.rcclAmdAdamW(None, 1, 7, 7, 7, 0, ctypes.byref(c), None) == ra.ncclInvalidArgument
    assert L.rcclAmdAdamW(None, -1, 7, 7, 7, 0, ctypes.byref(c), None) == ra.ncclInvalidArgument


def test_adamw_table_shape():
    _refused(lambda: ra.adamw(np.zeros((3, 7), dtype=np.int64), ra.ncclFloat32, ra.ncclFloat32, lr=1e-3, stream=0), "shape")
    _refused(lambda: ra.adamw(np.zeros((3, 8)), ra.ncclFloat32, ra.ncclFloat32, lr=1e-3, stream=0), "64-bit")
    assert ctypes.sizeof(ra.rcclAmdAdamWTensor_t) == 64


def test_sum_squares_refusals():
    need = ra.sum_squares_bytes(3)
    assert ra.sum_squares_bytes(0) == 0 and need >= 8 * 3
    call = lambda ptrs=(P,), counts=(5,), dt=ra.ncclFloat32, out=P, w=P: ra.sum_squares(np.array(ptrs), np.array(counts), dt, out, w, stream=0)  # noqa: E731
    for kw, text in ((dict(dt=ra.ncclInt32), "type"), (dict(out=None), "null"), (dict(out=P + 4), "misaligned"), (dict(w=P + 8), "misaligned"), (dict(w=None), "workspace"),
                     (dict(ptrs=(0,)), "null"), (dict(ptrs=(P + 2,)), "aligned"), (dict(counts=(2 ** 60,)), "elements"), (dict(counts=(5, 5)), "counts")):
        _refused(lambda: call(**kw), text)
    L = ra.lib()
    one = (ctypes.c_size_t * 1)(5)
    ptr = (ctypes.c_void_p * 1)(P)
    assert L.rcclAmdSumSquares(ptr, one, 1, ra.ncclFloat32, P, 0, P, ra.sum_squares_bytes(1) - 1, None) == ra.ncclInvalidArgument
    assert L.rcclAmdSumSquaresBytes(-1, ctypes.byref(ctypes.c_size_t())) == ra.ncclInvalidArgument
    assert L.rcclAmdSumSquaresBytes(1, None) == ra.ncclInvalidArgument


class _Tensor:
    """What the checks of a tensor ask, of one that lies on the current device."""
    def __init__(self, n, dtype):
        self.n, self.dtype = n, dtype

    def data_ptr(self):
        return P

    def numel(self):
        return self.n

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True


@pytest.mark.parametrize("counts", [[5], [], [5, 5, 5]])
def test_sum_squares_of_tensors_with_fewer_or_more_counts(counts, monkeypatch):
    """Two tensors and another number of counts: refused, no tensor is left out of the sum."""
    from rccl_amd import nccl
    monkeypatch.setattr(nccl, "_TORCH", {ra.ncclFloat32: "float32"})
    monkeypatch.setattr(nccl, "_current_device", lambda: 0)
    called = []
    monkeypatch.setattr(nccl.lib(), "rcclAmdSumSquares", lambda *a: called.append(a) or 0)
    call = lambda counts: ra.sum_squares([_Tensor(5, "float32")] * 2, counts, ra.ncclFloat32, P, P, stream=0)  # noqa: E731
    _refused(lambda: call(counts), "2 tensors with other counts")
    assert not called
    call([5, 5]), call(None)
    assert [a[2] for a in called] == [2, 2]


def test_sum_squares_of_no_tensors(monkeypatch):
    """A rank without tensors: its list is empty, and so need not be accompanied by counts."""
    from rccl_amd import nccl
    called = []
    monkeypatch.setattr(nccl.lib(), "rcclAmdSumSquares", lambda *a: called.append(a) or 0)
    for counts in (None, [], np.zeros(0, dtype=np.int64)):
        ra.sum_squares([], counts, ra.ncclFloat32, P, None, stream=0)
    assert [a[:3] for a in called] == [(None, None, 0)] * 3
    _refused(lambda: ra.sum_squares(np.array([P]), None, ra.ncclFloat32, P, P, stream=0), "counts")


def test_expert_sort_refusals():
    ok = dict(experts=P, expert_type=ra.ncclInt32, tokens=100, topk=8, first_expert=0, n_experts=16, row_align=1, position=P, source=P, offsets=P, counts=P, workspace=None, stream=0)
    for kw, text in ((dict(expert_type=ra.ncclFloat32), "expert type"), (dict(topk=0), "topk"), (dict(topk=65), "topk"), (dict(n_experts=0), "experts"), (dict(n_experts=1025), "experts"),
                     (dict(row_align=0), "rowAlign"), (dict(row_align=1025), "rowAlign"), (dict(first_expert=-1), "first expert"), (dict(first_expert=2 ** 63 - 1), "first expert"),
                     (dict(tokens=2 ** 28), "slots"), (dict(tokens=2 ** 62), "slots"), (dict(tokens=214748364, topk=10, n_experts=1024, row_align=1024), "rows"), (dict(experts=None), "null"),
                     (dict(position=None), "null"), (dict(experts=P + 2), "misaligned"), (dict(offsets=P + 1), "misaligned"), (dict(expert_type=ra.ncclInt64, experts=P + 4), "misaligned"),
                     (dict(tokens=100000), "workspace"), (dict(tokens=100000, workspace=P + 4), "misaligned")):
        _refused(lambda: ra.expert_sort(**{**ok, **kw}), text)
    assert ra.expert_sort_bytes(10, 8, 128) == 0
    assert ra.expert_sort_bytes(100000, 8, 128) >= 128 * 4
    assert ra.lib().rcclAmdExpertSortBytes(10, 8, 128, None) == ra.ncclInvalidArgument
    assert ra.expert_rows(10, 8, 4, 16) == 80 + 60


def test_row_operator_refusals():
    d = dict(x=P, out=2 * P, rows=64, datatype=ra.ncclBfloat16, tokens=8, topk=8, hidden=128, position=P, stream=0)
    for kw, text in ((dict(datatype=ra.ncclFloat64), "type"), (dict(topk=0), "topk"), (dict(topk=65), "topk"), (dict(hidden=0), "elements"), (dict(hidden=2 ** 31), "elements"),
                     (dict(rows=2 ** 31), "rows"), (dict(x_stride=127), "stride"), (dict(out_stride=127), "stride"), (dict(x_stride=2 ** 62), "stride"), (dict(x=None), "null"),
                     (dict(out=None), "null"), (dict(position=None), "null"), (dict(out=P), "same"), (dict(x=P + 1), "aligned"), (dict(position=P + 2), "aligned"),
                     (dict(offsets=P, n_experts=4), "together"), (dict(offsets=P, counts=P, n_experts=0), "experts"), (dict(tokens=2 ** 30), "slots")):
        _refused(lambda: ra.expert_dispatch(**{**d, **kw}), text)
    c = dict(z=P, rows=64, weights=P, weight_type=ra.ncclFloat32, y=2 * P, datatype=ra.ncclBfloat16, tokens=8, topk=8, hidden=128, position=P, stream=0)
    for kw, text in ((dict(weight_type=ra.ncclInt32), "weight type"), (dict(weights=P + 2), "aligned"), (dict(y=None), "null"), (dict(z=None), "null"), (dict(y=P), "same"), (dict(z_stride=1), "stride")):
        _refused(lambda: ra.expert_combine(**{**c, **kw}), text)
    b = dict(dy=P, z=2 * P, rows=64, weights=P, weight_type=ra.ncclFloat32, dz=3 * P, dweights=2 * P, datatype=ra.ncclBfloat16, tokens=8, topk=8, hidden=128, position=P, stream=0)
    for kw, text in ((dict(weight_type=-1), "weight type"), (dict(weights=None), "null"), (dict(dweights=None), "null"), (dict(z=None), "null"), (dict(dz=P), "overlaps"),
                     (dict(z=P), "overlaps"), (dict(dz=2 * P, dz_stride=256), "overlaps"), (dict(dweights=P), "same"), (dict(z_stride=3), "stride")):
        _refused(lambda: ra.expert_combine_backward(**{**b, **kw}), text)


def test_rows_without_work():
    ra.expert_dispatch(None, None, 0, ra.ncclFloat32, 0, 1, 8, None, stream=0)
    ra.expert_combine(None, 0, None, -1, None, ra.ncclFloat32, 0, 1, 8, None, stream=0)
    ra.expert_combine_backward(None, None, 0, None, ra.ncclFloat32, None, None, ra.ncclFloat32, 0, 1, 8, None, stream=0)


def test_the_mirror_module_leaves_what_is_not_plain():
    """Arguments that it does not take are answered with -1 (the long way then says what is wrong), wrong numbers of them with
    a TypeError; nothing is called."""
    from rccl_amd import _mirror as m
    for name, n in (("expert_sort", 13), ("expert_dispatch", 12), ("expert_combine", 11), ("expert_combine_backward", 16), ("sum_squares", 7), ("adamw", 18), ("expert_sort_bytes", 3), ("sum_squares_bytes", 1)):
        for junk in (None, "x", object(), -1, 2 ** 70, 1.5):
            assert getattr(m, name)(*[junk] * n) == -1, (name, junk)
        with pytest.raises(TypeError):
            getattr(m, name)()
    for args in ((), ({}, None, None, ()), ({}, None, None, (1,) * 7), ({}, None, None, ("x",) * 8), ({}, None, None, (0,) * 8), ([], None, None, (1,) * 8)):
        with pytest.raises((TypeError, ValueError)):
            m.bind(*args)


def test_without_the_mirror_module_calls_take_the_long_way(monkeypatch):
    """An interpreter that the module was not built for: one warning, and every call reaches the library's own checks."""
    import types
    import warnings
    from rccl_amd import nccl
    monkeypatch.setitem(sys.modules, "rccl_amd._mirror", None)               # (an import of it fails)
    monkeypatch.delattr(ra, "_mirror", raising=False)
    monkeypatch.setattr(nccl, "_mirror", None)
    s = types.SimpleNamespace(cuda_stream=0)
    row = np.array([[P, P, P, P, 0, 0, 0, 100]], dtype=np.int64)
    calls = [lambda: ra.adamw(row, ra.ncclFloat32, ra.ncclFloat32, lr=1e-3, step=0, stream=s),
             lambda: ra.sum_squares(np.array([P]), np.array([5]), ra.ncclInt32, P, P, stream=s),
             lambda: ra.expert_sort(P, ra.ncclInt32, 10, 65, 0, 16, 1, P, stream=s),
             lambda: ra.expert_dispatch(P, P, 64, ra.ncclFloat32, 8, 8, 128, P, stream=s),
             lambda: ra.expert_combine(P, 64, None, -1, P, ra.ncclFloat32, 8, 8, 128, P, stream=s),
             lambda: ra.expert_combine_backward(P, 2 * P, 64, P, ra.ncclFloat32, P, 2 * P, ra.ncclFloat32, 8, 8, 128, P, stream=s)]
    with pytest.warns(RuntimeWarning, match="_mirror"):
        _refused(calls[0], "first step")
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for call, text in zip(calls, ("first step", "type", "topk", "same", "same", "overlaps")):
            _refused(call, text)
        assert ra.sum_squares_bytes(0) == 0 and ra.expert_sort_bytes(100000, 8, 128) >= 128 * 4


def _make(tmp_path, python):
    """What make would run for a build from nothing."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rccl_amd", "csrc")
    r = subprocess.run(["make", "-n", "-C", csrc, f"PYTHON={python}", f"OUT={tmp_path}/lib.so", f"BUILD={tmp_path}/build"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert f"-o {tmp_path}/lib.so" in r.stdout
    return r.stdout


def test_the_library_is_built_without_python(tmp_path):
    """A host without an interpreter, or with one that has no headers, builds the library alone; others build the module too."""
    bare = tmp_path / "python"
    bare.write_text(f"#!/bin/sh\necho {tmp_path}/include\n")
    bare.chmod(0o755)
    for python in (str(tmp_path / "nothing"), str(bare)):
        out = _make(tmp_path, python)
        assert "without the module" in out and "mirror.c" not in out
    headers = os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h"))
    assert ("without the module" in _make(tmp_path, sys.executable)) == (not headers)
