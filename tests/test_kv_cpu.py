"""The paged key-value cache's C entries and torch ops without a GPU: arguments
are refused before any GPU work, workspaces have a size, shapes are inferred for
tracing, and the header's structs have the binding's layout."""
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
    p = _lib.KvPages(k=FAKE, v=FAKE, weights=FAKE, index=FAKE, num_pages=10, num_heads=2, page_size=16, head_dim=64,
                     dtype=_lib.DT_F16)
    for k, v in change.items():
        setattr(p, k, v)
    return p


def attend(**change):
    c = _lib.KvAttend(num_seqs=3, num_q_heads=4, dtype=_lib.DT_F16, q=FAKE, out=FAKE, block_tables=FAKE, table_stride=5,
                      max_pages=5, lengths=FAKE, scale=1.0, accumulate=1)
    for k, v in change.items():
        setattr(c, k, v)
    return c


def append(**change):
    c = _lib.KvAppend(num_tokens=3, slots=FAKE, dtype=_lib.DT_F16, k=FAKE, v=FAKE, q=FAKE, q_out=FAKE, num_q_heads=4,
                      positions=FAKE, cos_sin=FAKE, max_position=9, rot_dim=64, num_axes=1)
    c.sections[0] = 32
    for k, v in change.items():
        if k == "sections":
            c.sections[:] = v
        else:
            setattr(c, k, v)
    return c


def evict(**change):
    c = _lib.KvEvict(num_seqs=3, block_tables=FAKE, table_stride=5, max_pages=5, lengths=FAKE, new_lengths=FAKE, budget=7)
    for k, v in change.items():
        setattr(c, k, v)
    return c


BAD_PAGES = [{"num_pages": -1}, {"num_heads": 0}, {"page_size": 4}, {"page_size": 24}, {"page_size": 2048},
             {"head_dim": 0}, {"head_dim": 12}, {"head_dim": 264}, {"dtype": _lib.DT_F64}, {"dtype": _lib.DT_QI8_F32},
             {"k": None}, {"v": None}, {"k": FAKE + 8}, {"k_scale": FAKE}, {"dtype": _lib.DT_E4M3}]


def call(name, p, c):
    ref = [ctypes.byref(x) if x is not None else None for x in (p, c)]
    if name == "nve_amd_kv_append":
        return L.nve_amd_kv_append(*ref, None)
    return getattr(L, name)(*ref, None, 0, None)


@pytest.mark.parametrize("change", BAD_PAGES)
@pytest.mark.parametrize("name,make", [("nve_amd_kv_append", append), ("nve_amd_kv_attend", attend),
                                       ("nve_amd_kv_evict", evict)])
def test_bad_pages(name, make, change):
    assert call(name, pages(**change), make()) == _lib.INVALID_ARGUMENT
    assert _lib.last_error()


@pytest.mark.parametrize("name,make", [("nve_amd_kv_append", append), ("nve_amd_kv_attend", attend),
                                       ("nve_amd_kv_evict", evict)])
def test_null_structs(name, make):
    assert call(name, None, make()) == _lib.INVALID_ARGUMENT
    assert call(name, pages(), None) == _lib.INVALID_ARGUMENT


@pytest.mark.parametrize("change", [{"num_seqs": -1}, {"num_seqs": 1 << 20}, {"num_q_heads": 3}, {"num_q_heads": 0},
                                    {"dtype": _lib.DT_F32}, {"q": None}, {"out": None}, {"lengths": None},
                                    {"block_tables": None}, {"max_pages": -1}, {"max_pages": 1 << 40},
                                    {"max_length": -1}, {"scale": float("nan")}])
def test_bad_attend(change):
    assert call("nve_amd_kv_attend", pages(), attend(**change)) == _lib.INVALID_ARGUMENT


def test_attend_needs_weights_and_a_workspace():
    assert call("nve_amd_kv_attend", pages(weights=None), attend()) == _lib.INVALID_ARGUMENT
    assert call("nve_amd_kv_attend", pages(), attend()) == _lib.INVALID_ARGUMENT
    assert "orkspace" in _lib.last_error()
    n = ctypes.c_uint64()
    _lib.call("nve_amd_kv_attend_workspace_size", ctypes.byref(pages()), ctypes.byref(attend()), ctypes.byref(n))
    assert n.value >= 3 * 4 * 80 * 4  # a score per query head and slot
    need = n.value
    assert L.nve_amd_kv_attend(ctypes.byref(pages()), ctypes.byref(attend()), FAKE, need - 1, None) == _lib.INVALID_ARGUMENT
    assert L.nve_amd_kv_attend(ctypes.byref(pages()), ctypes.byref(attend()), FAKE + 4, need, None) == _lib.INVALID_ARGUMENT
    assert L.nve_amd_kv_attend_workspace_size(ctypes.byref(pages()), ctypes.byref(attend()), None) == _lib.INVALID_ARGUMENT


@pytest.mark.parametrize("change", [{"num_tokens": -1}, {"num_tokens": 1 << 40}, {"slots": None}, {"k": None},
                                    {"v": None}, {"q_out": None}, {"num_q_heads": -1}, {"dtype": _lib.DT_BF16},
                                    {"rot_dim": 63}, {"rot_dim": 66}, {"rot_dim": -2}, {"num_axes": 0}, {"num_axes": 5},
                                    {"positions": None}, {"cos_sin": None}, {"max_position": -1},
                                    {"sections": [31, 0, 0, 0]}, {"sections": [33, 0, 0, 0]},
                                    {"num_axes": 2, "sections": [33, -1, 0, 0]},
                                    {"num_axes": 2, "sections": [2**31 - 1, 2**31 - 1, 0, 0]}])
def test_bad_append(change):
    assert call("nve_amd_kv_append", pages(), append(**change)) == _lib.INVALID_ARGUMENT


@pytest.mark.parametrize("change", [{"num_seqs": -1}, {"num_seqs": 1 << 20}, {"lengths": None}, {"new_lengths": None},
                                    {"block_tables": None}, {"budget": -1}, {"sinks": -1}, {"recent": -1},
                                    {"max_pages": -1}])
def test_bad_evict(change):
    assert call("nve_amd_kv_evict", pages(), evict(**change)) == _lib.INVALID_ARGUMENT


def test_evict_needs_weights_index_and_a_workspace():
    for missing in ("weights", "index"):
        assert call("nve_amd_kv_evict", pages(**{missing: None}), evict()) == _lib.INVALID_ARGUMENT
    assert call("nve_amd_kv_evict", pages(), evict()) == _lib.INVALID_ARGUMENT
    assert "orkspace" in _lib.last_error()


@pytest.mark.parametrize("accumulate", [0, 1])
def test_attend_workspace_is_bounded_by_the_cache_and_by_the_tables(accumulate):
    """128 MiB of scores, or 4 for every slot there is, not one for every entry that the tables have room
    for; and none for the pages of a large cache that the tables cannot name."""
    def need(num_pages, seqs, max_pages):
        n = ctypes.c_uint64()
        p = pages(num_pages=num_pages, page_size=16, num_heads=8, head_dim=128)
        c = attend(num_seqs=seqs, num_q_heads=64, max_pages=max_pages, table_stride=max_pages, accumulate=accumulate)
        _lib.call("nve_amd_kv_attend_workspace_size", ctypes.byref(p), ctypes.byref(c), ctypes.byref(n))
        return n.value

    # rows, maxima and sums of the pieces: no more than of 8,192 pieces of 16 queries
    pieces = 8192 * 16 * (128 + 2) * 4 + (1 << 20)
    for max_pages in (16, 1024, 8192, 1 << 17):
        for num_pages in (2000, 50000):
            assert need(num_pages, 256, max_pages) <= pieces + accumulate * max(1 << 27, 4 * 64 * num_pages * 16 * 4)
    for num_pages in (100, 10000, 1 << 24):
        assert need(num_pages, 2, 50) <= pieces + accumulate * 2 * 64 * 1024 * 4


def test_more_heads_than_a_launch_has_workgroups():
    """A launch has fewer than 2^32 threads: 2^24 heads of sequences are refused, one less is not."""
    n = ctypes.c_uint64()
    p, c = pages(num_heads=1 << 9), attend(num_seqs=1 << 15, num_q_heads=1 << 9, max_pages=1)
    assert call("nve_amd_kv_attend", p, c) == _lib.INVALID_ARGUMENT
    assert "Too many heads" in _lib.last_error()
    c.num_seqs -= 1
    _lib.call("nve_amd_kv_attend_workspace_size", ctypes.byref(p), ctypes.byref(c), ctypes.byref(n))
    assert call("nve_amd_kv_append", pages(), append(num_tokens=1, num_q_heads=1 << 25)) == _lib.INVALID_ARGUMENT
    assert "num_q_heads" in _lib.last_error()


@pytest.mark.parametrize("offset", [0, 4, 8, -4, -8])
def test_evict_in_place_lengths_are_refused(offset):
    """A sequence's heads read its length while the first of them writes the new one."""
    refs = [ctypes.byref(pages()), ctypes.byref(evict(new_lengths=FAKE + offset))]
    assert L.nve_amd_kv_evict(*refs, FAKE, 1 << 20, None) == _lib.INVALID_ARGUMENT
    assert "overlap" in _lib.last_error()


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
@pytest.mark.parametrize("name,view", [("nve_amd_kv_pages_t", _lib.KvPages), ("nve_amd_kv_append_t", _lib.KvAppend),
                                       ("nve_amd_kv_attend_t", _lib.KvAttend), ("nve_amd_kv_evict_t", _lib.KvEvict)])
def test_struct_layout(tmp_path, name, view):
    fields = [f[0] for f in view._fields_]
    lines = "".join(f'printf("{f} %zu\\n", offsetof({name}, {f}));\n' for f in fields)
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "nve_amd_ext.h"\nint main(void) {{\n{lines}'
                   f'printf("size %zu\\n", sizeof({name}));\nreturn 0; }}\n')
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = dict(line.split() for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines())
    assert {f: int(got[f]) for f in fields} == {f: getattr(view, f).offset for f in fields}
    assert int(got["size"]) == ctypes.sizeof(view)


def test_shapes_are_inferred():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from pynve.torch import nve_kv

    with FakeTensorMode():
        q = torch.empty((3, 8, 64), dtype=torch.float16, device="cuda")
        p = torch.empty((5, 2, 16, 64), dtype=torch.float16, device="cuda")
        w = torch.empty((5, 2, 16), device="cuda")
        ix = torch.empty((5, 2, 16), dtype=torch.int32, device="cuda")
        t = torch.empty((3, 4), dtype=torch.int32, device="cuda")
        n = torch.empty(3, dtype=torch.int32, device="cuda")
        out, lse = nve_kv.kv_attend(q, p, p, t, n, return_lse=True)
        assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (3, 8) and lse.dtype == torch.float32
        assert nve_kv.kv_attend(q, p, p, t, n).shape == q.shape
        k = torch.empty((3, 2, 64), dtype=torch.float16, device="cuda")
        s = torch.empty(3, dtype=torch.int64, device="cuda")
        assert nve_kv.kv_append(k, k, p, p, s, q=q).shape == q.shape
        assert nve_kv.kv_append(k, k, p, p, s) is None
        assert nve_kv.kv_evict(p, p, w, ix, t, n, 8).shape == (3,)


def test_cpu_tensors_have_no_kernel():
    from pynve.torch import nve_kv

    p, q = torch.zeros((2, 1, 16, 8)), torch.zeros((1, 1, 8))
    with pytest.raises(NotImplementedError):
        nve_kv.kv_attend(q, p, p, torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32))
