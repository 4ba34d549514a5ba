"""Attention of one new token over the paged key-value cache (nve_ops::kv_attend)
against softmax attention in 64 bits: every type, head layouts, page sizes,
lengths around the kernels' tile sizes, long sequences, what lies past a length,
absent pages, strides, streams and graphs.  The bounds follow from the formula
(kv_reference.attend)."""
import math

import numpy as np
import pytest

import kv_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def setup(dtype, cache, lengths, q_heads, heads, dim, page, seed=0, spread=1.0, q_spread=1.0, extra=2, spare=3):
    rng = np.random.default_rng(seed)
    num_pages = sum(-(-n // page) for n in lengths) + spare
    k, ks = R.make_pages(cache, num_pages, heads, page, dim, rng, spread)
    v, vs = R.make_pages(cache, num_pages, heads, page, dim, rng)
    table = R.tables(lengths, page, num_pages, rng, extra)
    q = torch.from_numpy(rng.normal(0, q_spread, size=(len(lengths), q_heads, dim)).astype(np.float32))
    return {"q": q.to(R.TORCH[dtype]), "k": k, "v": v, "ks": ks, "vs": vs, "table": table,
            "lengths": np.asarray(lengths, np.int32), "dtype": dtype, "cache": cache, "page": page,
            "weights": torch.from_numpy(rng.random((num_pages, heads, page)).astype(np.float32))}


def poison_unused(s):
    """NaN and infinities in every row no sequence holds."""
    P, H, page, _ = s["k"].shape
    used = np.zeros((P, page), bool)
    for i, n in enumerate(s["lengths"]):
        _, p, o = R.slots_of(s["table"][i], int(n), page, P)
        used[p, o] = True
    free = ~torch.from_numpy(used)
    for name, bad in (("k", math.nan), ("v", math.inf)):
        x = s[name].to(torch.float32)
        x.transpose(1, 2)[free] = bad if s["cache"] != "e4m3" else math.nan
        s[name] = x.to(s[name].dtype)
    for name in ("ks", "vs"):
        if s[name] is not None:
            s[name].transpose(1, 2)[free] = math.inf


def cuda(x):
    return None if x is None else (torch.from_numpy(x) if isinstance(x, np.ndarray) else x).cuda()


def call(s, scale, accumulate=True, **kw):
    from pynve.torch import nve_kv

    w = cuda(s["weights"]) if accumulate else None
    out, lse = nve_kv.kv_attend(kw.pop("q", None) if "q" in kw else cuda(s["q"]), cuda(s["k"]), cuda(s["v"]),
                                cuda(s["table"]), cuda(s["lengths"]), scale=scale, k_scale=cuda(s["ks"]),
                                v_scale=cuda(s["vs"]), weights=w, return_lse=True, **kw)
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu(), None if w is None else w.cpu()


def check(s, scale, got, limit=None):
    out, lse, w = got
    lengths = s["lengths"] if limit is None else np.minimum(s["lengths"], limit)
    ro, rl, ra, bo, bl, ba = R.attend(s["q"], R.values64(s["k"], s["ks"]), R.values64(s["v"], s["vs"]), s["table"],
                                      lengths, scale, s["dtype"], s["cache"])
    err = np.abs(out.to(torch.float32).double().numpy() - ro)
    assert np.isfinite(err).all() and (err <= bo).all(), f"out: {np.max(err - bo)} over, {np.max(err)} off"
    empty = np.isneginf(rl)
    l64 = lse.double().numpy()
    assert np.array_equal(np.isneginf(l64), empty)
    assert (np.abs(l64 - rl)[~empty] <= bl[~empty]).all()
    if w is not None:
        w0 = s["weights"].double().numpy()
        touched = ra > 0
        e = np.abs(w.double().numpy() - (w0 + ra))
        assert (e[touched] <= (ba + 2.0**-23 * (w0 + ra))[touched]).all(), f"weights {np.nanmax(e[touched])} off"
        assert torch.equal(w[torch.from_numpy(~touched)], s["weights"][torch.from_numpy(~touched)])


TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "e4m3"), ("bf16", "e4m3")]


@pytest.mark.parametrize("q_heads,heads,dim,page", [(8, 2, 128, 16), (3, 3, 64, 8), (12, 1, 80, 32), (16, 2, 256, 64),
                                                    (10, 2, 8, 8), (20, 1, 96, 128), (34, 2, 136, 16), (7, 1, 40, 1024),
                                                    (70, 1, 128, 16)])
@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("accumulate", [False, True])
def test_types_and_layouts(dtype, cache, q_heads, heads, dim, page, accumulate):
    s = setup(dtype, cache, [0, 1, 9, 31, 32, 33, 64, 100, 257, 700], q_heads, heads, dim, page, seed=dim + page)
    poison_unused(s)
    check(s, dim**-0.5, call(s, dim**-0.5, accumulate))


@pytest.mark.parametrize("dim", [64, 128, 256, 56, 112, 248])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_widths_of_long_and_short_sequences(dtype, cache, accumulate, dim):
    """Every width the kernels are built for, whole and partly filled, over a few lengths beyond one workgroup's."""
    s = setup(dtype, cache, [3001, 40, 0, 1333, 5], 6, 2, dim, 16, seed=dim)
    poison_unused(s)
    check(s, dim**-0.5, call(s, dim**-0.5, accumulate))
    for i in range(5):  # the same through the path of short tables
        s["lengths"][i] = min(int(s["lengths"][i]), 500)
    s["table"] = np.ascontiguousarray(s["table"][:, :32])
    check(s, dim**-0.5, call(s, dim**-0.5, accumulate))


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_every_short_length(dtype, cache):
    s = setup(dtype, cache, list(range(0, 70)) + [127, 128, 129, 255, 256, 257, 511, 512, 513], 8, 2, 64, 16, seed=3)
    poison_unused(s)
    check(s, 0.125, call(s, 0.125))
    check(s, 0.125, call(s, 0.125, accumulate=False))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("lengths", [[20011], [5000, 1, 0, 16384, 16385, 3]])
def test_long_sequences(dtype, cache, lengths):
    """Few rows, long caches: the length is split and joined."""
    s = setup(dtype, cache, lengths, 8, 2, 64, 16, seed=11, q_spread=3.0)
    poison_unused(s)
    check(s, 0.125, call(s, 0.125))


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_many_sequences(dtype, cache):
    rng = np.random.default_rng(0)
    s = setup(dtype, cache, [int(n) for n in rng.integers(0, 90, size=300)], 4, 2, 64, 16, seed=12)
    check(s, 0.125, call(s, 0.125))


@pytest.mark.parametrize("dim", [64, 128, 256, 80])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_tables_far_longer_than_the_sequences(dtype, cache, accumulate, dim):
    """Tables of 131,072 slots over short sequences: the workgroups share the slots there are."""
    rng = np.random.default_rng(21)
    lengths = [int(n) for n in rng.integers(0, 40, size=95)] + [2500, 0, 777, 1, 1300]
    s = setup(dtype, cache, lengths, 6, 3, dim, 16, seed=22)
    wide = np.full((len(lengths), 8192), -1, np.int32)
    wide[:, :s["table"].shape[1]] = s["table"]
    s["table"] = wide
    poison_unused(s)
    check(s, dim**-0.5, call(s, dim**-0.5, accumulate))


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_weights_keep_their_bits(dtype, cache):
    """Values that cancel under the exact weights leave what the weights lost: all but 2^-22 of them is kept, 2^-17
    beside e4m3 values (of f32 statistics, D products added in f32, an exp2 and a sum)."""
    n, dim, scale = 200, 8, 0.35
    s = setup(dtype, cache, [4] * n, 2, 2, dim, 16, seed=33, q_spread=2.0**-6)
    q = s["q"].double().numpy()
    k = R.values64(s["k"], s["ks"])
    want, mass, size = np.zeros((n, 2, 1)), np.zeros((n, 2, 1)), np.zeros((n, 2, 1))
    for i in range(n):
        page = int(s["table"][i, 0])
        for h in range(2):
            x = scale * k[page, h, :4] @ q[i, h]
            w = np.exp(x - x.max())
            w /= w.sum()
            left = 0.0
            for t in range(4):  # the first value is 1, the others take back what the sum is so far
                v = 1.0 if t == 0 else -left / w[t]
                if cache == "e4m3":
                    s["v"][page, h, t] = math.copysign(1.0, v)
                    s["vs"][page, h, t] = abs(v)
                    v = math.copysign(float(s["vs"][page, h, t]), v)
                else:
                    s["v"][page, h, t] = v
                    v = float(s["v"][page, h, t, 0])
                left += w[t] * v
                mass[i, h] += w[t] * abs(v)
            want[i, h], size[i, h] = left, scale * (np.abs(k[page, h, :4]) @ np.abs(q[i, h])).max()
    out = call(s, scale)[0].double().numpy()
    rel = 2 * (dim + 8) * 2.0**-24 * size + 2.0**-20 + 2.0**-23 * math.log2(5) + (2.0**-17 if cache == "e4m3" else 2.0**-22)
    bound = rel * mass * 1.01 + R.HALF_ULP[dtype] * np.maximum(np.abs(want) + rel * mass, R.SMALL[dtype])
    err = np.abs(out - want)
    assert (err <= bound).all(), f"{(err / bound).max()} times the bound"


@pytest.mark.parametrize("dtype,cache", TYPES[:3])
@pytest.mark.parametrize("length", [1, 30, 700, 5000])
@pytest.mark.parametrize("sign", [1, -1])
def test_infinite_values(dtype, cache, length, sign):
    """An infinity among the values is the output in its column, as in the formula; both signs give NaN there."""
    s = setup(dtype, cache, [length, length], 4, 2, 64, 16, seed=31)
    s["q"] *= 0.25  # no weight below 2^-38 of the largest
    at = np.random.default_rng(32).integers(0, length, size=3)
    for i, (where, d) in enumerate(zip(at, (3, 40, 63))):
        s["v"][int(s["table"][0, where // 16]), :, int(where) % 16, d] = sign * math.inf * (-1) ** i
    both = length > 1
    if both:
        a, b = 0, length - 1
        s["v"][int(s["table"][0, a // 16]), :, a % 16, 20] = math.inf
        s["v"][int(s["table"][0, b // 16]), :, b % 16, 20] = -math.inf
    out, lse, w = call(s, 0.125)
    assert torch.isfinite(lse).all() and torch.isfinite(w).all()
    for i, d in enumerate((3, 40, 63)):
        assert (out[0, :, d] == sign * math.inf * (-1) ** i).all(), d
    if both:
        assert torch.isnan(out[0, :, 20]).all()
    other = torch.ones(64, dtype=torch.bool)
    other[[3, 40, 63] + [20] * both] = False
    finite = {**s, "v": torch.nan_to_num(s["v"], posinf=0.0, neginf=0.0)}
    clean = call(finite, 0.125)
    assert torch.equal(out[0][:, other], clean[0][0][:, other]) and torch.equal(out[1], clean[0][1])
    check(finite, 0.125, clean)


@pytest.mark.parametrize("dim", [8, 56, 192, 248])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_partly_filled_widths_in_tables_far_longer(dtype, cache, accumulate, dim):
    """The kernels for up to 64 and up to 256 values with narrower rows, their workgroups sharing the slots there are."""
    rng = np.random.default_rng(29)
    lengths = [int(n) for n in rng.integers(0, 40, size=95)] + [2500, 0, 777, 1, 1300]
    s = setup(dtype, cache, lengths, 6, 3, dim, 16, seed=30)
    wide = np.full((len(lengths), 8192), -1, np.int32)
    wide[:, :s["table"].shape[1]] = s["table"]
    s["table"] = wide
    poison_unused(s)
    check(s, dim**-0.5, call(s, dim**-0.5, accumulate))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("length,width", [(0, 1 << 20), (1, 131072), (100, 131072), (777, 1 << 20), (4000, 131072),
                                          (20011, 1 << 20)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_one_sequence_in_a_wide_table(dtype, cache, length, width, accumulate):
    """Pieces by the sequence's length: the result of a table that fits, bit for bit."""
    s = setup(dtype, cache, [length], 6, 2, 64, 16, seed=28, extra=1)
    poison_unused(s)
    wide = {**s, "table": np.full((1, width // 16), -1, np.int32)}
    wide["table"][:, :s["table"].shape[1]] = s["table"]
    got = call(wide, 0.125, accumulate)
    check(s, 0.125, got)
    if length > 512:
        for a, b in zip(got, call(s, 0.125, accumulate)):
            assert a is b is None or torch.equal(a, b)


def test_one_sequence_takes_no_longer_in_a_wide_table():
    """32,000 slots in a table of 2^20, on as many workgroups as in a table that fits (it took 10 times as long on
    the few pieces that the table's width gave them)."""
    from pynve.torch import nve_kv

    pages = 2000
    k = torch.randn((pages, 8, 16, 128), device="cuda").half()
    v, q = torch.randn_like(k), torch.randn((1, 32, 128), device="cuda").half()
    length = torch.tensor([pages * 16], dtype=torch.int32, device="cuda")
    tight = torch.randperm(pages, device="cuda").int().view(1, -1)
    wide = torch.full((1, 1 << 16), -1, dtype=torch.int32, device="cuda")
    wide[:, :pages] = tight

    def time(table):
        best = math.inf
        for _ in range(5):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            nve_kv.kv_attend(q, k, v, table, length)
            start.record()
            for _ in range(20):
                nve_kv.kv_attend(q, k, v, table, length)
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end))
        return best

    assert time(wide) < 4 * time(tight)


@pytest.mark.parametrize("page", [8, 32])
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_weights_in_tables_wider_than_the_cache(dtype, cache, page):
    """Tables of 32,768 slots, 60 sequences of 40 query heads in pieces: the weights' scores lie by the cache's slots."""
    rng = np.random.default_rng(24)
    s = setup(dtype, cache, [2100, 3, 1500, 0, 1, 700] + [int(n) for n in rng.integers(0, 40, size=54)], 40, 2, 64, page,
              seed=25)
    wide = np.full((60, 32768 // page), -1, np.int32)
    wide[:, :s["table"].shape[1]] = s["table"]
    s["table"] = wide
    s["table"][0, 7], s["table"][2, 1] = -1, s["k"].shape[0]
    poison_unused(s)
    check(s, 0.125, call(s, 0.125))


@pytest.mark.parametrize("dtype,cache", [("f16", "f16"), ("f32", "f32")])
def test_weights_of_many_short_sequences_in_wide_tables(dtype, cache):
    """A workgroup a unit, scores by slot (2,100 sequences) and in order (half of them): the same bits."""
    rng = np.random.default_rng(26)
    s = setup(dtype, cache, [int(n) for n in rng.integers(0, 60, size=2100)], 32, 2, 64, 16, seed=27)
    wide = np.full((2100, 16 if dtype == "f32" else 32), -1, np.int32)
    wide[:, :s["table"].shape[1]] = s["table"]
    s["table"] = wide
    if dtype == "f32":  # a workgroup a unit up to 256 slots
        for n in ("q", "table", "lengths"):
            s[n] = np.concatenate([s[n]] * 2) if n != "q" else torch.cat([s[n]] * 2)
        s["lengths"][2100:] = 0
    out, lse, w = call(s, 0.125)
    n = len(s["lengths"]) // 2
    w2 = s["weights"]
    for part in (slice(0, n), slice(n, 2 * n)):
        h = {**s, "q": s["q"][part], "table": np.ascontiguousarray(s["table"][part]), "lengths": s["lengths"][part],
             "weights": w2}
        o2, l2, w2 = call(h, 0.125)
        assert torch.equal(out[part], o2) and torch.equal(lse[part], l2)
    assert torch.equal(w, w2) and not torch.equal(w, s["weights"])


@pytest.mark.parametrize("dtype,cache", [("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("q_heads", [34, 40])
def test_wide_groups_in_long_tables(dtype, cache, q_heads):
    """More than 16 query heads a key head, sequences in several pieces, both ways of sharing the work."""
    s = setup(dtype, cache, [2100, 3, 1500, 0] + [5] * 96, q_heads, 1, 64, 16, seed=23)
    check(s, 0.125, call(s, 0.125))
    wide = np.full((100, 8192), -1, np.int32)
    wide[:, :s["table"].shape[1]] = s["table"]
    s["table"] = wide
    check(s, 0.125, call(s, 0.125))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("accumulate", [False, True])
def test_one_slot_is_copied(dtype, cache, accumulate):
    """A softmax over one slot is 1: the output is the value row itself."""
    s = setup(dtype, cache, [1, 1, 1], 6, 3, 128, 16, seed=4, q_spread=30.0)
    out, lse, w = call(s, 0.2, accumulate)
    for i in range(3):
        v = R.values64(s["v"], s["vs"])[s["table"][i, 0], :, 0].astype(np.float32)
        want = torch.from_numpy(np.repeat(v, 2, axis=0)).to(R.TORCH[dtype])
        if cache == "e4m3":  # the scale meets the weight before the code does: 16 bits of it are kept
            assert (out[i].float() - want.float()).abs().max() <= want.float().abs().max() * (2.0**-15 + R.HALF_ULP[dtype] * 2)
        else:
            assert torch.equal(out[i], want)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_wide_scores(dtype, cache):
    """Scores of some hundreds: one slot takes nearly all the weight, most of the others none."""
    s = setup(dtype, cache, [1000, 37, 4097], 8, 2, 64, 16, seed=5, spread=4.0, q_spread=8.0)
    check(s, 1.0, call(s, 1.0))


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_flat_tail_is_not_lost(dtype, cache):
    """One slot far above 20,000 equal ones that together weigh as much: 2e4 e^-10 = 0.91."""
    s = setup(dtype, cache, [20001], 2, 1, 64, 16, seed=6)
    q = torch.zeros_like(s["q"])
    q[..., 0] = 1.0
    k = torch.zeros(s["k"].shape)
    top = (int(s["table"][0, 700]), 0, 3)
    k[top][0] = 10.0
    if cache == "e4m3":
        s["ks"] = torch.ones_like(s["ks"])
    s["q"], s["k"] = q, k.to(s["k"].dtype)
    check(s, 1.0, call(s, 1.0))


@pytest.mark.parametrize("dtype,cache", TYPES[:3])
def test_scores_of_minus_infinity(dtype, cache):
    """-infinity scores weigh nothing; where there are no others the row is empty."""
    s = setup(dtype, cache, [50, 600, 33], 4, 2, 64, 16, seed=7)
    s["q"][..., 0] = 1.0
    for i, n in enumerate(s["lengths"]):
        _, p, o = R.slots_of(s["table"][i], int(n), 16, s["k"].shape[0])
        off = np.arange(n) >= 0 if i == 2 else np.arange(n) % 40 < 35
        s["k"][torch.from_numpy(p[off]), :, torch.from_numpy(o[off]), 0] = -math.inf
    out, lse, w = call(s, 0.3)
    assert torch.equal(out[2], torch.zeros_like(out[2]))
    check(s, 0.3, (out, lse, w))


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_absent_pages(dtype, cache):
    """Page numbers outside the cache inside a length: their slots are left out."""
    s = setup(dtype, cache, [300, 17, 40], 4, 2, 64, 16, seed=8)
    s["table"][0, 3], s["table"][0, 7], s["table"][0, 18] = -1, s["k"].shape[0], 2**31 - 1
    s["table"][1, :] = -5
    check(s, 0.125, call(s, 0.125))


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_length_bounds(dtype, cache):
    """Negative lengths count as 0, those above the table (or max_length) as that bound."""
    s = setup(dtype, cache, [64, 48, 5], 4, 2, 64, 16, seed=9, extra=0)
    full = call(s, 0.125, max_length=64)
    check(s, 0.125, full)
    s["lengths"] = np.asarray([2**31 - 1, 48, -7], np.int32)
    got = call(s, 0.125)
    s["lengths"] = np.asarray([64, 48, 0], np.int32)
    check(s, 0.125, got)
    check(s, 0.125, call(s, 0.125, max_length=33), limit=33)


def test_no_sequences_and_no_pages():
    s = setup("f16", "f16", [], 4, 2, 64, 16)
    assert call(s, 0.125)[0].shape == (0, 4, 64)
    s = setup("f16", "f16", [0, 0], 4, 2, 64, 16, extra=0, spare=0)
    out, lse, _ = call(s, 0.125)
    assert torch.equal(out, torch.zeros_like(out)) and torch.isneginf(lse).all()


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_strides(dtype, cache):
    """q as a slice of a wider projection at an odd element offset; a block table wider than it is read."""
    s = setup(dtype, cache, [100, 31, 450], 6, 2, 72, 8, seed=10)
    base = torch.zeros((3, 9, 75), dtype=s["q"].dtype)
    base[:, 1:7, 3:75] = s["q"]
    out, lse, w = call(s, 0.1, q=base.cuda()[:, 1:7, 3:75])
    check(s, 0.1, (out, lse, w))
    wide = cuda(s["table"]).repeat(1, 2)
    from pynve.torch import nve_kv

    again = nve_kv.kv_attend(cuda(s["q"]), cuda(s["k"]), cuda(s["v"]), wide[:, :s["table"].shape[1]],
                             cuda(s["lengths"]), scale=0.1, k_scale=cuda(s["ks"]), v_scale=cuda(s["vs"]))
    assert torch.equal(again.cpu(), out)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_the_same_every_time(dtype, cache):
    s = setup(dtype, cache, [3000, 20, 9000], 8, 2, 128, 16, seed=13)
    a, b = call(s, 0.1), call(s, 0.1)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_rows_past_32_bits():
    """Pages whose elements lie past 2^31 of the cache's start."""
    from pynve.torch import nve_kv

    heads, page, dim = 8, 16, 128
    num_pages = 2**31 // (heads * page * dim) + 40
    k = torch.zeros((num_pages, heads, page, dim), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    s = setup("f16", "f16", [500], 8, heads, dim, page, seed=14)
    n = s["k"].shape[0]
    k[-n:], v[-n:] = s["k"].cuda(), s["v"].cuda()
    table = cuda(s["table"])
    table = torch.where(table >= 0, table + num_pages - n, table)
    w = torch.zeros((num_pages, heads, page), device="cuda")
    w[-n:] = s["weights"].cuda()
    out, lse = nve_kv.kv_attend(cuda(s["q"]), k, v, table, cuda(s["lengths"]), scale=0.1, weights=w, return_lse=True)
    check(s, 0.1, (out.cpu(), lse.cpu(), w[-n:].cpu()))


def test_another_stream():
    """Inputs made on one stream, used on another that waits for it."""
    from pynve.torch import nve_kv

    s = setup("bf16", "bf16", [4000, 900], 8, 2, 128, 16, seed=15)
    want = call(s, 0.1)
    side = torch.cuda.Stream()
    args = [cuda(s[n]) for n in ("q", "k", "v", "table", "lengths")]
    w = cuda(s["weights"])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = nve_kv.kv_attend(*args, scale=0.1, weights=w, return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), want[0]) and torch.equal(lse.cpu(), want[1]) and torch.equal(w.cpu(), want[2])


def test_graph_replays():
    """Captured once, replayed over new queries and lengths, each replay against the eager call."""
    from pynve.torch import nve_kv

    s = setup("f16", "f16", [3000, 1500, 64], 8, 2, 64, 16, seed=16)
    q, k, v, table, lengths = (cuda(s[n]) for n in ("q", "k", "v", "table", "lengths"))
    w = torch.zeros(s["weights"].shape, device="cuda")
    nve_kv.kv_attend(q, k, v, table, lengths, scale=0.125, weights=w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nve_kv.kv_attend(q, k, v, table, lengths, scale=0.125, weights=w)
    for i in range(4):
        q.copy_(torch.randn(q.shape, device="cuda"))
        lengths.copy_(torch.tensor([3000 - 700 * i, 1500 - i, 16 * i], dtype=torch.int32))
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        w2 = torch.zeros_like(w)
        want = nve_kv.kv_attend(q, k, v, table, lengths, scale=0.125, weights=w2)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(w, w2)


def test_refusals():
    from pynve.torch import nve_kv

    s = setup("f16", "f16", [20, 5], 4, 2, 64, 16)
    base = {n: cuda(s[n]) for n in ("q", "k", "v", "table", "lengths")}

    def run(**change):
        kw = {n: change.pop(n) for n in ("k_scale", "v_scale", "weights", "max_length", "scale") if n in change}
        a = {**base, **change}
        return nve_kv.kv_attend(a["q"], a["k"], a["v"], a["table"], a["lengths"], **kw)

    run()
    bad_values = [{"q": base["q"][:, :3]}, {"q": base["q"][:1]}, {"q": base["q"][..., :56]}, {"q": base["q"][0]},
                  {"q": base["q"].transpose(1, 2)}, {"q": base["q"].cpu()}, {"table": base["table"][:1]},
                  {"table": base["table"].cpu()}, {"lengths": base["lengths"][:1]}, {"v": base["v"][:2]},
                  {"k": base["k"].transpose(1, 2)}, {"weights": torch.zeros(3, device="cuda")}, {"max_length": -1},
                  {"scale": math.nan}, {"k_scale": cuda(s["weights"]), "v_scale": cuda(s["weights"])},
                  {"k": base["k"][:, :, :4].contiguous(), "v": base["v"][:, :, :4].contiguous()},
                  {"k": base["k"][:, :, :12].contiguous(), "v": base["v"][:, :, :12].contiguous()},
                  {"k": base["k"][..., :60].contiguous(), "v": base["v"][..., :60].contiguous(), "q": base["q"][..., :60]},
                  {"k": base["k"].to(torch.float8_e4m3fn), "v": base["v"].to(torch.float8_e4m3fn)},
                  {"q": base["q"].float()}]
    for change in bad_values:
        with pytest.raises(ValueError):
            run(**change)
    for change in [{"table": base["table"].long()}, {"lengths": base["lengths"].long()}, {"q": base["q"].double()},
                   {"k": base["k"].float()}, {"weights": cuda(s["weights"]).half()}]:
        with pytest.raises((TypeError, ValueError)):
            run(**change)
    with pytest.raises(RuntimeError, match="gradient"):
        run(q=base["q"].clone().requires_grad_())
    with torch.no_grad():
        run(q=base["q"].clone().requires_grad_())
