"""The microscaled operators without a GPU: the C ABI's symbols and host-only answers, refusals, and the 64-bit oracle
against hand-worked values."""
from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from cs464_b200 import _abi, build, micro
from oracle import micro as om

HEADER = Path(__file__).resolve().parent.parent / "include" / "b2g_micro.h"


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = set(re.findall(r"\b(b2g_micro_[a-z0-9_]+)\s*\(", text))
    assert names == set(_abi.MICRO_EXPORTS)
    _abi.load()
    out = subprocess.run(["nm", "-D", "--defined-only", str(build.LIB_PATH)], capture_output=True, text=True).stdout
    assert names <= set(re.findall(r" T (b2g_[a-z0-9_]+)$", out, flags=re.M))


def test_source_hash_covers_the_gemm_family_only():
    """Stored winners name the GEMM sources: a change to the microscaled operators alone must not invalidate them."""
    assert build.source_hash() != build.build_hash()
    seen = [f for f in build.sources() if f.name.startswith("b2g_")]
    assert {f.name for f in seen} == {"b2g_forest.cu", "b2g_gemm.cu", "b2g_timing.cu"}
    assert any(f.name.startswith("micro_") for f in build.sources())


@pytest.mark.parametrize("fmt,rows,cols,pitch,scales", [
    ("mxfp8", 1, 1, 32, 512), ("mxfp8", 128, 128, 128, 512), ("mxfp8", 129, 129, 160, 2048),
    ("mxfp4", 1, 33, 32, 512), ("nvfp4", 300, 4096, 2048, 3 * 64 * 512), ("nvfp4", 0, 64, 32, 0), ("mxfp4", 5, 0, 0, 0),
])
def test_layout(fmt, rows, cols, pitch, scales):
    p, s = ctypes.c_int64(), ctypes.c_int64()
    rc = _abi.load().b2g_micro_layout(micro.FORMATS[fmt], rows, cols, ctypes.byref(p), ctypes.byref(s))
    assert rc == 0 and (p.value, s.value) == (pitch, scales)
    assert micro._layout(micro.FORMATS[fmt], rows, cols) == (pitch, scales)


def _tensor(fmt=1, rows=4, cols=64, codes=4096, pitch=64, scales=8192, scale=None):
    return _abi.MicroTensor(fmt, 0, rows, cols, codes, pitch, scales, scale)


@pytest.mark.parametrize("bad,text", [
    (dict(fmt=0), "format"), (dict(fmt=4), "format"), (dict(rows=-1), "negative"), (dict(cols=1 << 31), "dimension_too_large"),
    (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(codes=4097), "aligned"), (dict(scales=8200), "aligned"),
    (dict(pitch=32), "pitch"), (dict(pitch=80), "pitch"), (dict(fmt=3, pitch=32), "scale"),
])
def test_entry_points_refuse_bad_tensors(bad, text):
    """Each refusal comes from the host's checks, before any launch: the addresses here are never read."""
    lib = _abi.load()
    t, ok = _tensor(**bad), _tensor()
    mat = _abi.MicroMatrix(4096, 64, 1)
    calls = [lambda: lib.b2g_micro_quantize(mat, _abi.VALUE_BF16, t, None),
             lambda: lib.b2g_micro_dequantize(t, mat, _abi.VALUE_BF16, None),
             lambda: lib.b2g_micro_matmul(t, ok, 4096, 64, _abi.VALUE_BF16, None, None),
             lambda: lib.b2g_micro_matmul(ok, t, 4096, 64, _abi.VALUE_BF16, None, None),
             lambda: lib.b2g_micro_rms_norm(mat, None, 4096, None, None, t, 4, 64, 1e-5, _abi.VALUE_BF16, None),
             lambda: lib.b2g_micro_silu_mul(mat, None, t, 4, 64, _abi.VALUE_BF16, None)]
    for c in calls:
        assert c() in (_abi.B2G_ERR_INVALID_ARG, _abi.B2G_ERR_UNSUPPORTED)
        assert text in _abi.last_error()


def test_entry_points_refuse_bad_arguments():
    lib = _abi.load()
    a, mat = _tensor(), _abi.MicroMatrix(4096, 64, 1)
    inv = _abi.B2G_ERR_INVALID_ARG
    assert lib.b2g_micro_matmul(a, _tensor(fmt=2, pitch=32), 4096, 64, 1, None, None) == _abi.B2G_ERR_UNSUPPORTED
    assert _abi.last_error().startswith("format_mismatch")
    assert lib.b2g_micro_matmul(a, _tensor(cols=32), 4096, 64, 1, None, None) == inv       # K differs
    assert lib.b2g_micro_matmul(a, a, 4096, 64, _abi.VALUE_F32, None, None) == inv         # fp32 output
    assert lib.b2g_micro_matmul(a, a, None, 64, 1, None, None) == inv
    assert lib.b2g_micro_matmul(a, a, 4096, 3, 1, None, None) == inv                       # ldc < N
    assert lib.b2g_micro_quantize(None, 1, a, None) == inv and lib.b2g_micro_quantize(mat, 3, a, None) == inv
    assert lib.b2g_micro_plan_create(a, a, 4096, 64, 1, None, None) == inv
    assert lib.b2g_micro_plan_launch(None, None) == inv and lib.b2g_micro_plan_destroy(None) == 0
    assert lib.b2g_micro_rms_norm(mat, None, 4096, None, mat, a, 4, 64, 1e-5, 1, None) == inv   # two outputs
    assert lib.b2g_micro_rms_norm(mat, None, 4096, None, None, None, 4, 64, 1e-5, 1, None) == inv
    assert lib.b2g_micro_rms_norm(mat, None, 4096, mat, mat, None, 4, 64, 1e-5, 1, None) == inv  # h without a residual
    assert lib.b2g_micro_rms_norm(mat, None, 4096, None, None, a, 5, 64, 1e-5, 1, None) == inv  # q of other rows
    assert lib.b2g_micro_rms_norm(mat, None, 4096, None, mat, None, 4, 64, 1e-5, 2, None) == inv
    assert lib.b2g_micro_rms_norm_backward(mat, mat, 4096, None, mat, 4096, 4096, 0, 4, 64, 1e-5, 1,
                                           None) == _abi.B2G_ERR_WORKSPACE
    assert lib.b2g_micro_silu_mul(mat, None, None, 4, 64, 1, None) == inv
    assert lib.b2g_micro_silu_mul_backward(mat, None, mat, 4, 64, 1, None) == inv
    assert lib.b2g_micro_tensor_scale(mat, 4, 64, 1, None, None) == inv
    n = ctypes.c_size_t()
    assert lib.b2g_micro_matmul_values_workspace(3, 130, 5, 70, ctypes.byref(n)) == 0
    assert n.value == 32 + 135 * micro._layout(3, 1, 70)[0] + micro._layout(3, 130, 70)[1] + micro._layout(3, 5, 70)[1]
    assert lib.b2g_micro_matmul_values_workspace(0, 4, 4, 4, ctypes.byref(n)) == inv
    assert lib.b2g_micro_matmul_values(mat, mat, 4, 4, 4, 1, 1, 4096, 4, 1, None, 0, None, None) == _abi.B2G_ERR_WORKSPACE
    assert lib.b2g_micro_matmul_values(mat, mat, 4, 4, 4, 1, 1, 4096, 3, 1, 4096, 1 << 20, None, None) == inv
    assert lib.b2g_micro_matmul_values(mat, mat, 4, 4, 4, 1, 7, 4096, 4, 1, 4096, 1 << 20, None, None) == inv
    assert lib.b2g_micro_rms_norm_workspace(4, 64, ctypes.byref(n)) == 0 and n.value >= 64 * 4  # an fp32 row at least
    assert lib.b2g_micro_rms_norm_workspace(-1, 64, ctypes.byref(n)) == inv


def test_norm_refuses_columns_past_its_counters():
    """A row's columns are counted in 31 bits, a round of up to 4096 past its end included."""
    lib = _abi.load()
    for cols in (2 ** 31 - 8191, 2 ** 31 - 200, 2 ** 31, 2 ** 32 + 64):
        mat = _abi.MicroMatrix(4096, cols, 1)
        assert lib.b2g_micro_rms_norm(mat, mat, 4096, mat, mat, None, 1, cols, 1e-5, 1, None) == _abi.B2G_ERR_UNSUPPORTED
        assert _abi.last_error().startswith("dimension_too_large")
        assert lib.b2g_micro_rms_norm_backward(mat, mat, 4096, None, mat, 4096, 4096, 1 << 50, 1, cols, 1e-5, 1,
                                               None) == _abi.B2G_ERR_UNSUPPORTED


def test_gate_refuses_columns_past_its_counters():
    """A row's eight-column chunks are counted in 32 bits, those of a whole block of 256 threads past its end included."""
    lib = _abi.load()
    for cols in (2 ** 35 - 2047, 2 ** 35, 2 ** 36 + 64):
        mat = _abi.MicroMatrix(4096, 0, 0)
        for rc in (lib.b2g_micro_silu_mul(mat, mat, None, 1, cols, 1, None),
                   lib.b2g_micro_silu_mul_backward(mat, mat, mat, 1, cols, 1, None)):
            assert rc == _abi.B2G_ERR_UNSUPPORTED and _abi.last_error().startswith("dimension_too_large")


def test_empty_calls_do_nothing():
    lib = _abi.load()
    e = _tensor(rows=0, codes=None, scales=None)
    mat = _abi.MicroMatrix(None, 64, 1)
    assert lib.b2g_micro_quantize(mat, 1, e, None) == 0
    assert lib.b2g_micro_dequantize(e, mat, 1, None) == 0
    assert lib.b2g_micro_matmul(e, _tensor(), None, 64, 1, None, None) == 0
    assert lib.b2g_micro_rms_norm(mat, None, None, None, mat, None, 0, 64, 1e-5, 1, None) == 0
    assert lib.b2g_micro_silu_mul(mat, mat, None, 4, 0, 1, None) == 0


def test_python_refuses_cpu_tensors_and_bad_formats():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="no CPU path"):
        micro.quantize(x, "mxfp8")
    with pytest.raises(ValueError, match="format must be one of mxfp8, mxfp4, nvfp4"):
        micro.quantize(x, "fp8")
    with pytest.raises(ValueError, match="no CPU path"):
        micro.MicroTensor(x.byte(), x.byte(), (4, 64), "mxfp8")
    for call in (lambda: micro.rms_norm(x, x[0]), lambda: micro.silu_mul(x), lambda: micro.micro_linear(x, x),
                 lambda: micro.rms_norm_backward(x, x, x[0]), lambda: micro.silu_mul_backward(x, x)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
    with pytest.raises(TypeError, match="MicroTensors"):
        micro.micro_matmul(x, x)
    with pytest.raises(TypeError, match="MicroTensors"):
        micro.micro_mlp(x, None, x[0], x, x)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        micro.MicroMatmul(torch.float32)


def test_a_tensors_fields_cannot_be_assigned():
    """The kernels read the addresses, sizes and format packed when the tensor was made: an assignment that they would not
    see (and that could drop the only owner of a scale they go on reading) is refused."""
    q = object.__new__(micro.MicroTensor)
    for field in ("scale", "shape", "format", "codes", "scales", "device"):
        with pytest.raises(AttributeError):
            setattr(q, field, None)


def test_fake_tensors_leave_nothing_behind(monkeypatch):
    """Under a mode that replaces tensors (torch's tracing) calls raise, and what the module keeps per device is not made of
    replaced tensors: real calls would go on using them, a status word at address 0 among them."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from cs464_b200.matmul import status_word
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(micro, "_get_device", lambda: 0)
    monkeypatch.setattr(micro, "_raw_stream", lambda index: 0)
    kept = micro._BYTES, micro._STATUS_AT, status_word.__globals__["_STATUS"]
    before = [dict(d) for d in kept]
    try:
        for d in kept:
            d.clear()
        with FakeTensorMode():
            x = torch.empty(4, 64, dtype=torch.bfloat16, device="cuda")
            for call in (lambda: micro.rms_norm(x, x[0], format="mxfp8"), lambda: micro.quantize(x), lambda: micro._status(0)):
                with pytest.raises(RuntimeError):
                    call()
        assert not any(kept)
    finally:
        for d, b in zip(kept, before):
            d.clear()
            d.update(b)


def test_dependents_are_launched_after_the_tensor_memory_is_allocated():
    """A dependent's CTA holds tensor memory while it waits for the whole grid before it. Were it let in while a CTA of that
    grid still waits for columns, the two could wait for each other for good, so the signal has to stand after the
    allocation in every kernel that has one, and nowhere else."""
    for f in sorted(build.CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", f.read_text())
        kernels = re.split(r"\b__global__\b", text)[1:]
        for k in kernels:
            allocations = [m.start() for m in re.finditer(r"\btmem_alloc(?:_pair)?\(", k)]
            signals = [m.start() for m in re.finditer(r"launch_dependents", k)]
            assert bool(signals) == bool(allocations), f.name
            assert not signals or min(signals) > max(allocations), f.name
    asm = [f.name for f in sorted(build.CSRC.iterdir()) if "griddepcontrol.launch_dependents" in f.read_text()]
    assert asm == ["b2g_ptx.cuh"]


def test_wait_limit_refusals():
    lib = _abi.load()
    assert lib.b2g_micro_plan_wait_limit(None, 5) == _abi.B2G_ERR_INVALID_ARG and "null plan" in _abi.last_error()
    e, plan = _tensor(rows=0, codes=None, scales=None), ctypes.c_void_p()
    assert lib.b2g_micro_plan_create(e, _tensor(), None, 64, 1, None, ctypes.byref(plan)) == 0
    assert lib.b2g_micro_plan_wait_limit(plan, -1) == _abi.B2G_ERR_INVALID_ARG and "wait_limit_us" in _abi.last_error()
    assert lib.b2g_micro_plan_wait_limit(plan, 5) == 0  # an empty product: nothing waits
    assert lib.b2g_micro_plan_destroy(plan) == 0


# ---------------------------------------------------------------- the oracle
def test_oracle_codes_by_hand():
    x = np.zeros((1, 64))
    x[0, :9] = [6.0, 0.25, 0.75, -2.5, 5.0, 3.5, 1.75, -0.26, 1.25]
    x[0, 32] = 6.0001
    x[0, 33] = 6.0
    c, s = om.quantize(x, "mxfp4")
    # ties go to the even code: .25 -> 0, .75 -> 1, -2.5 -> -2, 5 -> 4, 3.5 -> 4, 1.75 -> 2, 1.25 -> 1
    assert list(c[0, :9]) == [7, 0, 2, 8 + 4, 6, 6, 4, 8 + 1, 2]
    assert list(s[0]) == [127, 128]                      # 6 fits scale 1; 6.0001 needs 2
    assert list(c[0, 32:34]) == [5, 5]                   # 3.00005 -> 3, 3 -> 3
    c, s = om.quantize(np.array([[448.0, 449.0, 1.0, -17.0]]), "mxfp8")
    assert s[0, 0] == 128 and om.values(c, s, "mxfp8")[0].tolist() == [448.0, 448.0, 1.0, -16.0]
    c, s = om.quantize(np.array([[1.0, np.inf], [np.nan, 2.0], [0.0, -0.0]]), "mxfp8")
    assert list(s[:, 0]) == [255, 255, 0]
    assert np.isnan(om.values(c, s, "mxfp8")[:2]).all() and (om.values(c, s, "mxfp8")[2] == 0).all()


def test_oracle_nvfp4_by_hand():
    assert om.tensor_scale(np.array([[2688.0]])) == 1.0 and om.tensor_scale(np.array([[2689.0]])) == 2.0
    assert om.tensor_scale(np.array([[np.inf, 1.3125]])) == 2.0 ** -11 and om.tensor_scale(np.zeros((1, 1))) == 2.0 ** -100
    c, s = om.quantize(np.array([[12.0, 5.0, -24.0]]), "nvfp4", 1.0)  # 24 / 6 = 4: an e4m3 value
    assert om.values(c, s, "nvfp4", 1.0)[0].tolist() == [12.0, 4.0, -24.0]  # 5 / 4 = 1.25 ties to the even code, 1
    c, s = om.quantize(np.array([[1e6, -3.0]]), "nvfp4", 1.0)         # past 2688: saturates
    assert om.values(c, s, "nvfp4", 1.0)[0].tolist() == [2688.0, -0.0]
    c, s = om.quantize(np.array([[1e-4, 5e-5]]), "nvfp4", 1.0)        # 1e-4 / 6 rounds to a scale of zero
    assert s[0, 0] == 0 and (om.values(c, s, "nvfp4", 1.0) == 0).all()


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4", "nvfp4"])
def test_oracle_layout_matches_the_header(fmt):
    """Scale byte (row, block) lies where include/b2g_micro.h says; codes pack the lower column in the low bits."""
    rows, cols = 200, 700
    rng = np.random.default_rng(0)
    block = om.BLOCK[fmt]
    n = -(-cols // block)
    kt = -(-n // 4)
    table = rng.integers(1, 100, (rows, n), dtype=np.uint8)
    raw = np.zeros(-(-rows // 128) * kt * 512, np.uint8)
    for r in range(rows):
        for b in range(n):
            raw[((r // 128) * kt + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4] = table[r, b]
    pitch = -(-cols // 32) * (32 if fmt == "mxfp8" else 16)
    codes = np.zeros((rows, pitch), np.uint8)
    codes[3, 5] = 0x21
    c, s, zero = om.unpack(codes, raw, rows, cols, fmt)
    assert zero and (s == table).all()
    assert c[3, 5] == 0x21 if fmt == "mxfp8" else (c[3, 10], c[3, 11]) == (1, 2)
