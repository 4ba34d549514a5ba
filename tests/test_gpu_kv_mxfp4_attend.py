"""Attention over pages of 4-bit values against softmax attention in 64 bits on the values that the
codes stand for: types, head layouts, widths, lengths, split and shared launches, what lies past a
length, NaN scales, absent pages, strides, streams and graphs.  Bounds: kv_reference.attend."""
import math

import numpy as np
import pytest

import kv4_reference as R4
import kv_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def setup(dtype, lengths, q_heads, heads, dim, page, seed=0, spread=1.0, q_spread=1.0, extra=2, spare=3):
    rng = np.random.default_rng(seed)
    num_pages = sum(-(-n // page) for n in lengths) + spare
    k, ks = R4.make_pages(num_pages, heads, page, dim, rng, spread)
    v, vs = R4.make_pages(num_pages, heads, page, dim, rng)
    q = torch.from_numpy(rng.normal(0, q_spread, size=(len(lengths), q_heads, dim)).astype(np.float32))
    return {"q": q.to(R.TORCH[dtype]), "k": k, "v": v, "ks": ks, "vs": vs, "dtype": dtype, "page": page,
            "table": R.tables(lengths, page, num_pages, rng, extra), "lengths": np.asarray(lengths, np.int32),
            "weights": torch.from_numpy(rng.random((num_pages, heads, page)).astype(np.float32))}


def poison_unused(s):
    """Codes of all kinds and NaN scales in every row no sequence holds."""
    P, H, page, _ = s["k"].shape
    used = np.zeros((P, page), bool)
    for i, n in enumerate(s["lengths"]):
        _, p, o = R.slots_of(s["table"][i], int(n), page, P)
        used[p, o] = True
    free = ~torch.from_numpy(used)
    for name in ("k", "v"):
        s[name].transpose(1, 2)[free] = 0xf7
        s[name + "s"].transpose(1, 2)[free] = 255


def cuda(x):
    return None if x is None else (torch.from_numpy(x) if isinstance(x, np.ndarray) else x).cuda()


def pages(s):
    (k, ks), (v, vs) = R4.typed(cuda(s["k"]), cuda(s["ks"])), R4.typed(cuda(s["v"]), cuda(s["vs"]))
    return k, v, {"k_scale": ks, "v_scale": vs}


def call(s, scale, accumulate=True, **kw):
    from pynve.torch import nve_kv

    w = cuda(s["weights"]) if accumulate else None
    k, v, scales = pages(s)
    out, lse = nve_kv.kv_attend(cuda(s["q"]), k, v, cuda(s["table"]), cuda(s["lengths"]), scale=scale, weights=w,
                                return_lse=True, **scales, **kw)
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu(), None if w is None else w.cpu()


def check(s, scale, got):
    out, lse, w = got
    ro, rl, ra, bo, bl, ba = R.attend(s["q"], R4.values64(s["k"], s["ks"]), R4.values64(s["v"], s["vs"]), s["table"],
                                      s["lengths"], scale, s["dtype"], "mxfp4")
    # exp2's results below 2^-126 are 0: a slot may lose that much of a weight
    bo += 2.0**-126 * np.maximum(s["lengths"], 0)[:, None, None] * np.nanmax(np.abs(R4.values64(s["v"], s["vs"])))
    err = np.abs(out.to(torch.float32).double().numpy() - ro)
    assert np.isfinite(err).all() and (err <= bo).all(), f"out: {np.max(err - bo)} over, {np.max(err)} off"
    empty = np.isneginf(rl)
    l64 = lse.double().numpy()
    assert np.array_equal(np.isneginf(l64), empty)
    assert (np.abs(l64[~empty] - rl[~empty]) <= bl[~empty]).all()
    if w is not None:
        w0 = s["weights"].double().numpy()
        touched = ra > 0
        e = np.abs(w.double().numpy() - (w0 + ra))
        assert (e[touched] <= (ba + 2.0**-23 * (w0 + ra))[touched]).all(), f"weights {np.nanmax(e[touched])} off"
        assert torch.equal(w[torch.from_numpy(~touched)], s["weights"][torch.from_numpy(~touched)])


DTYPES = ["f16", "bf16"]


@pytest.mark.parametrize("q_heads,heads,dim,page", [(8, 2, 128, 16), (3, 3, 64, 8), (12, 1, 96, 32), (16, 2, 256, 64),
                                                    (10, 2, 32, 8), (20, 1, 160, 128), (34, 2, 224, 16),
                                                    (7, 1, 64, 1024), (70, 1, 128, 16), (17, 17, 192, 16)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("accumulate", [False, True])
def test_types_and_layouts(dtype, q_heads, heads, dim, page, accumulate):
    s = setup(dtype, [0, 1, 9, 31, 32, 33, 64, 100, 257, 700], q_heads, heads, dim, page, seed=dim + page)
    poison_unused(s)
    check(s, dim**-0.5, call(s, dim**-0.5, accumulate))


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 256])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_widths_of_long_and_short_sequences(dtype, accumulate, dim):
    s = setup(dtype, [3001, 40, 0, 1333, 5], 6, 2, dim, 16, seed=dim)
    poison_unused(s)
    check(s, dim**-0.5, call(s, dim**-0.5, accumulate))
    for i in range(5):  # the same through the path of short tables
        s["lengths"][i] = min(int(s["lengths"][i]), 500)
    s["table"] = np.ascontiguousarray(s["table"][:, :32])
    check(s, dim**-0.5, call(s, dim**-0.5, accumulate))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_short_length(dtype, dim):
    s = setup(dtype, list(range(0, 70)) + [127, 128, 129, 255, 256, 257, 511, 512, 513], 8, 2, dim, 16, seed=3)
    poison_unused(s)
    check(s, 0.125, call(s, 0.125))
    check(s, 0.125, call(s, 0.125, accumulate=False))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths", [[20011], [5000, 1, 0, 16384, 16385, 3]])
def test_long_sequences(dtype, lengths):
    s = setup(dtype, lengths, 8, 2, 128, 16, seed=11, q_spread=3.0)
    poison_unused(s)
    check(s, 0.1, call(s, 0.1))


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_sequences(dtype):
    rng = np.random.default_rng(0)
    s = setup(dtype, [int(n) for n in rng.integers(0, 90, size=300)], 4, 2, 64, 16, seed=12)
    check(s, 0.125, call(s, 0.125))


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_tables_far_longer_than_the_sequences(dtype, accumulate, dim):
    """Tables of 131,072 slots over short sequences: the workgroups share the slots there are."""
    rng = np.random.default_rng(21)
    lengths = [int(n) for n in rng.integers(0, 40, size=95)] + [2500, 0, 777, 1, 1300]
    s = setup(dtype, lengths, 6, 3, dim, 16, seed=22)
    wide = np.full((len(lengths), 8192), -1, np.int32)
    wide[:, :s["table"].shape[1]] = s["table"]
    s["table"] = wide
    poison_unused(s)
    check(s, dim**-0.5, call(s, dim**-0.5, accumulate))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_scores_keep_the_queries_bits(dtype, dim):
    """Queries whose large values meet zeros and whose small ones, 2^-14 below, decide; groups of 32 far apart in size."""
    s = setup(dtype, [300, 37, 5000], 4, 2, dim, 16, seed=41)
    big = torch.arange(dim) % 32 == 5
    q = s["q"].float()
    q[..., big] *= 2.0**7
    q[..., ~big] *= 2.0**-3
    s["q"] = q.to(R.TORCH[dtype])
    codes = s["k"]
    at = torch.arange(dim // 2) % 16 == 2  # value 5 of 32 is the high half of byte 2
    codes[..., at] = codes[..., at] & 0x0f
    s["ks"] += torch.from_numpy(np.random.default_rng(42).integers(-2, 6, size=tuple(s["ks"].shape)).astype(np.uint8))
    check(s, 1.0, call(s, 1.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_every_code_and_scale(dtype, dim):
    """All bytes of codes under exponents from far below to far above one; one slot, so that the output is its value."""
    n = 40
    s = setup(dtype, [1] * n, 2, 1, dim, 16, seed=43)
    rng = np.random.default_rng(44)
    s["v"] = torch.from_numpy(rng.integers(0, 256, size=tuple(s["v"].shape)).astype(np.uint8))
    s["vs"] = torch.from_numpy(rng.integers(127 - 30, 127 + 13, size=tuple(s["vs"].shape)).astype(np.uint8))
    check(s, 0.01, call(s, 0.01))
    if dtype == "bf16":
        s["vs"] = torch.from_numpy(rng.integers(5, 251, size=tuple(s["vs"].shape)).astype(np.uint8))
        check(s, 0.01, call(s, 0.01))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", [1, 30, 700, 5000])
def test_nan_scales(dtype, length):
    """A NaN among the values is NaN in its 32 columns alone; one among the keys is its whole row."""
    s = setup(dtype, [length, length], 4, 2, 128, 16, seed=31)
    want = call(s, 0.1)
    where = length // 2
    s["vs"][int(s["table"][0, where // 16]), 1, where % 16, 2] = 255
    out, lse, _ = call(s, 0.1)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, 2:, 64:96] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], want[0][~bad]) and torch.equal(lse, want[1])
    s["ks"][int(s["table"][1, where // 16]), 0, where % 16, 1] = 255
    out, lse, _ = call(s, 0.1)
    assert torch.isnan(out[1, :2]).all() and torch.equal(out[1, 2:], want[0][1, 2:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_absent_pages(dtype):
    s = setup(dtype, [200, 90, 40], 4, 2, 64, 16, seed=5)
    s["table"][0, 3], s["table"][0, 12], s["table"][1, 0], s["table"][2, :] = -1, 10**6, -5, -1
    check(s, 0.125, call(s, 0.125))


def test_strides_and_no_pages():
    from pynve.torch import nve_kv

    s = setup("bf16", [300, 50], 6, 3, 64, 16, seed=6)
    want = call(s, 0.1)
    k, v, scales = pages(s)
    q = torch.zeros((2, 9, 67), dtype=torch.bfloat16, device="cuda")
    q[:, 2:8, 3:] = s["q"].cuda()
    table = torch.zeros((2, 3 + s["table"].shape[1]), dtype=torch.int32, device="cuda")
    table[:, 3:] = cuda(s["table"])
    got = nve_kv.kv_attend(q[:, 2:8, 3:], k, v, table[:, 3:], cuda(s["lengths"]), scale=0.1, **scales)
    assert torch.equal(got.cpu(), want[0])
    none = {n: t[:0] for n, t in scales.items()}
    out, lse = nve_kv.kv_attend(q[:, 2:8, 3:], k[:0], v[:0], table, cuda(s["lengths"]), return_lse=True, **none)
    assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_scales_at_any_byte(dim):
    from pynve.torch import nve_kv

    s = setup("f16", [300, 50], 4, 2, dim, 16, seed=8)
    want = call(s, 0.1)
    k, v, scales = pages(s)
    for n in ("k_scale", "v_scale"):
        x = scales[n].view(torch.uint8)
        apart = torch.zeros(x.numel() + 3, dtype=torch.uint8, device="cuda")[3:].view(x.shape)
        scales[n] = apart.copy_(x).view(torch.float8_e8m0fnu)
        assert scales[n].data_ptr() % 4 == 3
    w = cuda(s["weights"])
    out = nve_kv.kv_attend(cuda(s["q"]), k, v, cuda(s["table"]), cuda(s["lengths"]), scale=0.1, weights=w, **scales)
    assert torch.equal(out.cpu(), want[0]) and torch.equal(w.cpu(), want[2])


def test_max_length_bounds_the_lengths():
    s = setup("f16", [500, 700], 4, 2, 128, 16, seed=7)
    got = call(s, 0.1, max_length=400)
    s["lengths"] = np.minimum(s["lengths"], 400)
    check(s, 0.1, got)


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_same_every_time(dtype):
    s = setup(dtype, [3000, 20, 9000], 8, 2, 128, 16, seed=13)
    a, b = call(s, 0.1), call(s, 0.1)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_rows_past_32_bits():
    """Pages whose bytes lie past 2^32 of the cache's start."""
    from pynve.torch import nve_kv

    heads, page, dim = 8, 64, 128
    num_pages = 2**32 // (heads * page * dim // 2) + 40
    s = setup("bf16", [500], 8, heads, dim, page, seed=14)
    n = s["k"].shape[0]
    full = {}
    for name in ("k", "v", "ks", "vs"):
        x = s[name]
        full[name] = torch.zeros((num_pages, *x.shape[1:]), dtype=torch.uint8, device="cuda")
        full[name][-n:] = x.cuda()
    (k, ks), (v, vs) = R4.typed(full["k"], full["ks"]), R4.typed(full["v"], full["vs"])
    table = cuda(s["table"])
    table = torch.where(table >= 0, table + num_pages - n, table)
    w = torch.zeros((num_pages, heads, page), device="cuda")
    w[-n:] = s["weights"].cuda()
    out, lse = nve_kv.kv_attend(cuda(s["q"]), k, v, table, cuda(s["lengths"]), scale=0.1, k_scale=ks, v_scale=vs,
                                weights=w, return_lse=True)
    check(s, 0.1, (out.cpu(), lse.cpu(), w[-n:].cpu()))


def test_another_stream_and_graph_replays():
    from pynve.torch import nve_kv

    s = setup("f16", [3000, 1500, 64], 8, 2, 128, 16, seed=16)
    want = call(s, 0.1)
    k, v, scales = pages(s)
    q, table, lengths, w = (cuda(s[n]) for n in ("q", "table", "lengths", "weights"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = nve_kv.kv_attend(q, k, v, table, lengths, scale=0.1, weights=w, **scales)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), want[0]) and torch.equal(w.cpu(), want[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nve_kv.kv_attend(q, k, v, table, lengths, scale=0.1, weights=w, **scales)
    for i in range(4):
        q.copy_(torch.randn(q.shape, device="cuda"))
        lengths.copy_(torch.tensor([3000 - 700 * i, 1500 - i, 16 * i], dtype=torch.int32))
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        w2 = torch.zeros_like(w)
        again = nve_kv.kv_attend(q, k, v, table, lengths, scale=0.1, weights=w2, **scales)
        torch.cuda.synchronize()
        assert torch.equal(out, again) and torch.equal(w, w2)


def test_refusals():
    from pynve.torch import nve_kv

    s = setup("f16", [20, 5], 4, 2, 64, 16)
    k, v, scales = pages(s)
    base = {"q": cuda(s["q"]), "k": k, "v": v, "table": cuda(s["table"]), "lengths": cuda(s["lengths"]), **scales}

    def run(**change):
        a = {**base, **change}
        return nve_kv.kv_attend(a["q"], a["k"], a["v"], a["table"], a["lengths"], k_scale=a["k_scale"],
                                v_scale=a["v_scale"])

    run()
    raw = lambda t: t.view(torch.uint8)  # noqa: E731
    for change in [{"k_scale": None}, {"v_scale": None}, {"k_scale": scales["k_scale"][..., :1]},
                   {"k_scale": raw(scales["k_scale"])[:2].view(torch.float8_e8m0fnu)}, {"q": base["q"][..., :32]},
                   {"q": base["q"].float()}, {"v_scale": raw(scales["v_scale"]).cpu().view(torch.float8_e8m0fnu)},
                   {"k": raw(k)[..., :24].contiguous().view(k.dtype), "v": raw(v)[..., :24].contiguous().view(k.dtype),
                    "q": base["q"][..., :48]}]:
        with pytest.raises(ValueError):
            run(**change)
    for change in [{"k": raw(k), "v": raw(v)}, {"k_scale": raw(scales["k_scale"])},
                   {"k_scale": torch.zeros(k.shape[:3], device="cuda")}, {"v": raw(v)}]:
        with pytest.raises(TypeError):
            run(**change)
