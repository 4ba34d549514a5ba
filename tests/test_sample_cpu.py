"""Token sampling without a GPU: arguments are refused before any GPU work, the header's struct has the
binding's layout, shapes are inferred for tracing, and the tests' own restatement gives known answers."""
import ctypes
import math
import os
import shutil
import subprocess

import numpy as np
import pytest

import sample_reference as R
from pynve import _lib

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
L = _lib.load()
FAKE = 1 << 20  # an aligned address that no refused call reads


def call(**change):
    c = _lib.Sample(**{**dict(num_rows=3, vocab_size=50, dtype=_lib.DT_F32, logits=FAKE, row_stride=50, u=FAKE,
                              temperature=1.0, top_p=1.0, tokens=FAKE), **change})
    return L.nve_amd_sample(ctypes.byref(c), FAKE, 1 << 40, None)


@pytest.mark.parametrize("change", [{"num_rows": -1}, {"num_rows": 1 << 40}, {"vocab_size": 0}, {"vocab_size": 1 << 31},
                                    {"dtype": _lib.DT_F64}, {"dtype": _lib.DT_E4M3}, {"dtype": _lib.DT_XMXFP4},
                                    {"logits": None}, {"u": None}, {"tokens": None}, {"temperature": -1.0},
                                    {"temperature": math.nan}, {"top_k": -1}, {"top_p": -1.0}, {"top_p": math.nan},
                                    {"min_p": -1.0}, {"min_p": 2.0}, {"min_p": math.nan}])
def test_refusals(change):
    assert call(**change) == _lib.INVALID_ARGUMENT
    assert _lib.last_error()


def test_null_struct_and_workspace():
    assert L.nve_amd_sample(None, None, 0, None) == _lib.INVALID_ARGUMENT
    n = ctypes.c_uint64()
    c = _lib.Sample(num_rows=3, vocab_size=50000, dtype=_lib.DT_F32, logits=FAKE, row_stride=50000, u=FAKE, temperature=1.0,
                    top_p=1.0, tokens=FAKE)
    assert L.nve_amd_sample_workspace_size(ctypes.byref(c), None) == _lib.INVALID_ARGUMENT
    _lib.call("nve_amd_sample_workspace_size", ctypes.byref(c), ctypes.byref(n))
    if n.value:
        for ws, size in ((None, n.value), (FAKE, n.value - 1), (FAKE + 4, n.value)):
            assert L.nve_amd_sample(ctypes.byref(c), ws, size, None) == _lib.INVALID_ARGUMENT
            assert "orkspace" in _lib.last_error()


@pytest.mark.parametrize("rows", [1, 64, 256, 300, 1024, 2048, 5000, 1 << 20])
@pytest.mark.parametrize("vocab", [16, 2049, 16384, 32003, 65536, 65537, 131072, 1 << 19, 1 << 30])
@pytest.mark.parametrize("dtype", [_lib.DT_F32, _lib.DT_F16, _lib.DT_BF16])
def test_workspace_is_bounded(dtype, vocab, rows):
    """2^27 logits at once at most, 4 bytes for 64 of them (2^25, for 16), 12 for 1,024, and 2,048 histograms of 16 KiB."""
    n = ctypes.c_uint64()
    c = _lib.Sample(num_rows=rows, vocab_size=vocab, dtype=dtype, logits=FAKE, row_stride=vocab, u=FAKE, temperature=1.0,
                    top_p=0.9, tokens=FAKE)
    _lib.call("nve_amd_sample_workspace_size", ctypes.byref(c), ctypes.byref(n))
    assert n.value <= (8 << 20) + (12 << 17) + (32 << 20) + (1 << 20)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_struct_layout(tmp_path):
    fields = [f[0] for f in _lib.Sample._fields_]
    lines = "".join(f'printf("{f} %zu\\n", offsetof(nve_amd_sample_t, {f}));\n' for f in fields)
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "nve_amd_ext.h"\nint main(void) {{\n{lines}'
                   'printf("size %zu\\n", sizeof(nve_amd_sample_t));\nreturn 0; }\n')
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = dict(line.split() for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines())
    assert {f: int(got[f]) for f in fields} == {f: getattr(_lib.Sample, f).offset for f in fields}
    assert int(got["size"]) == ctypes.sizeof(_lib.Sample)


def test_shapes_are_inferred_and_cpu_tensors_have_no_kernel():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from pynve.torch.nve_sample import sample_tokens

    with FakeTensorMode():
        out = sample_tokens(torch.empty((3, 9), device="cuda"), torch.empty(3, device="cuda"), top_k=2)
        assert out.shape == (3,) and out.dtype == torch.int64
    with pytest.raises(NotImplementedError):
        sample_tokens(torch.zeros(1, 4), torch.zeros(1))


def test_the_restatement():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    pick = lambda u, **k: R.sample_row(x, u, **k)  # noqa: E731
    assert [pick(u) for u in (0.0, 0.09, 0.11, 0.49, 0.51, 0.69, 0.71, 1.0)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert [pick(u, top_k=2) for u in (0.0, 0.57, 0.58)] == [1, 1, 3]
    assert [pick(u, top_p=0.5) for u in (0.0, 0.57, 0.58)] == [1, 1, 3] and pick(0.9, top_p=0.39) == 1
    assert [pick(u, min_p=0.45) for u in (0.0, 0.44, 0.45, 0.66, 0.67)] == [1, 1, 2, 2, 3]
    assert pick(0.99, temperature=0.0) == 1 and R.sample_row([1.0, 2.0, 2.0], 0.9, top_k=1) == 1
    assert R.sample_row([-math.inf, math.nan], 0.5) == -1 and R.sample_row([0.0, math.inf], 0.0) == 1
