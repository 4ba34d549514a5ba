"""4-bit pages and normed appends without a GPU: arguments are refused before any GPU work, shapes are
inferred for tracing, and the header's struct has the binding's layout."""
import ctypes
import os
import shutil
import subprocess

import pytest

from pynve import _lib

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
L = _lib.load()
FAKE = 1 << 20  # an aligned address that no refused call reads


def pages(**change):
    return _lib.KvPages(**{**dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, weights=FAKE, index=FAKE, num_pages=10,
                                  num_heads=2, page_size=16, head_dim=64, dtype=_lib.DT_XMXFP4), **change})


def append(**change):
    c = _lib.KvAppend(**{**dict(num_tokens=3, slots=FAKE, dtype=_lib.DT_F16, k=FAKE, v=FAKE, q=FAKE, q_out=FAKE,
                                num_q_heads=4, positions=FAKE, cos_sin=FAKE, max_position=9, rot_dim=64, num_axes=1),
                         **change})
    c.sections[0] = 32
    return c


def attend(**change):
    return _lib.KvAttend(**{**dict(num_seqs=3, num_q_heads=4, dtype=_lib.DT_F16, q=FAKE, out=FAKE, block_tables=FAKE,
                                   table_stride=5, max_pages=5, lengths=FAKE, scale=1.0), **change})


def evict():
    return _lib.KvEvict(num_seqs=3, block_tables=FAKE, table_stride=5, max_pages=5, lengths=FAKE, new_lengths=FAKE + 64,
                        budget=7)


def norm(**change):
    return _lib.KvNorm(**{**dict(q_weight=FAKE, k_weight=FAKE, eps=1e-6), **change})


def call(p, c, n=None):
    a = [ctypes.byref(p), ctypes.byref(c)]
    if isinstance(c, _lib.KvAppend):
        return L.nve_amd_kv_append(*a, None) if n is None else L.nve_amd_kv_append_norm(*a, ctypes.byref(n), None)
    return (L.nve_amd_kv_attend if isinstance(c, _lib.KvAttend) else L.nve_amd_kv_evict)(*a, None, 0, None)


@pytest.mark.parametrize("change", [{"head_dim": 48}, {"head_dim": 8}, {"head_dim": 288}, {"k_scale": None},
                                    {"v_scale": None}, {"k": None}, {"v": FAKE + 8}, {"page_size": 12}, {"dtype": 35},
                                    {"page_size": 1024, "num_heads": 65535, "head_dim": 128}])
@pytest.mark.parametrize("make", [append, attend, evict])
def test_bad_pages(make, change):
    assert call(pages(**change), make()) == _lib.INVALID_ARGUMENT
    assert _lib.last_error()


@pytest.mark.parametrize("make", [append, attend])
@pytest.mark.parametrize("dtype", [_lib.DT_F32, _lib.DT_E4M3, _lib.DT_XMXFP4])
def test_rows_of_16_bits_alone(make, dtype):
    assert call(pages(), make(dtype=dtype)) == _lib.INVALID_ARGUMENT
    assert "float16 or bfloat16" in _lib.last_error()


@pytest.mark.parametrize("change", [{"eps": -1e-9}, {"eps": float("nan")}, {"eps": float("inf")}])
def test_bad_norms(change):
    for p in (pages(), pages(dtype=_lib.DT_F16, k_scale=None, v_scale=None)):
        assert call(p, append(), norm(**change)) == _lib.INVALID_ARGUMENT
        assert "eps" in _lib.last_error()
        assert call(p, append(q=None), norm()) == _lib.INVALID_ARGUMENT
        assert "q_weight" in _lib.last_error()
    assert L.nve_amd_kv_append_norm(ctypes.byref(pages()), ctypes.byref(append()), None, None) == _lib.INVALID_ARGUMENT
    assert L.nve_amd_kv_append_norm(None, ctypes.byref(append()), ctypes.byref(norm()), None) == _lib.INVALID_ARGUMENT


def test_the_4_bit_type_is_no_row_format_of_a_table():
    """Lookups and caches of rows refuse it, as every type they do not know."""
    st = L.nve_amd_find_and_pool(0, 1, FAKE, FAKE, 1, 64, _lib.DT_XMXFP4, 0, 0, None, 0, 0, None, 0, _lib.DT_F32, FAKE, 64,
                                 0, 0, None)
    assert st == _lib.INVALID_ARGUMENT


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_struct_layout(tmp_path):
    fields = [f[0] for f in _lib.KvNorm._fields_]
    lines = "".join(f'printf("{f} %zu\\n", offsetof(nve_amd_kv_norm_t, {f}));\n' for f in fields)
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "nve_amd_ext.h"\nint main(void) {{\n{lines}'
                   'printf("size %zu\\n", sizeof(nve_amd_kv_norm_t));\nreturn NVE_DTYPE_X_MXFP4 != 34; }\n')
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = dict(line.split() for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines())
    assert {f: int(got[f]) for f in fields} == {f: getattr(_lib.KvNorm, f).offset for f in fields}
    assert int(got["size"]) == ctypes.sizeof(_lib.KvNorm)


def test_a_cache_of_4_bits_has_its_shapes():
    from pynve.torch import nve_kv

    c = nve_kv.KVCache(5, 3, 96, page=8, dtype=torch.float4_e2m1fn_x2, device="cpu")
    assert c.k.shape == c.v.shape == (5, 3, 8, 48) and c.k.dtype == torch.float4_e2m1fn_x2
    assert c.k_scale.shape == c.v_scale.shape == (5, 3, 8, 3) and c.k_scale.dtype == torch.float8_e8m0fnu
    with pytest.raises(ValueError):
        nve_kv.KVCache(5, 3, 80, dtype=torch.float4_e2m1fn_x2, device="cpu")


def test_shapes_are_inferred():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from pynve.torch import nve_kv

    with FakeTensorMode():
        q = torch.empty((3, 8, 64), dtype=torch.float16, device="cuda")
        k = torch.empty((3, 2, 64), dtype=torch.float16, device="cuda")
        w = torch.empty(64, dtype=torch.float16, device="cuda")
        s = torch.empty(3, dtype=torch.int64, device="cuda")
        p = torch.empty((5, 2, 16, 64), dtype=torch.float16, device="cuda")
        assert nve_kv.kv_append(k, k, p, p, s, q=q, q_norm=w, k_norm=w).shape == q.shape
        assert nve_kv.kv_append(k, k, p, p, s, k_norm=w) is None
