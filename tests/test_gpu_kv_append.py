"""New tokens entering the paged key-value cache (nve_ops::kv_append): rotated
queries and keys, written rows, e4m3 codes and scales, bit for bit what the
definition's f32 steps give (kv_reference.rotate, kv_reference.quantize), and
near the rotation in 64 bits; what is not written stays."""
import numpy as np
import pytest

import kv_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "e4m3"), ("bf16", "e4m3")]


def bits(t):
    return t.contiguous().view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def table_of(positions, rot, seed=0):
    a = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(0, rot, 2) / max(rot, 1))
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


def run(dtype, cache, tokens, q_heads, heads, dim, page, rot=0, sections=None, interleaved=False, seed=0, fused=False,
        bad_slots=False, bad_positions=False, index=True, track=True, special=False, with_q=True):
    from pynve.torch import nve_kv

    rng = np.random.default_rng(seed)
    num_pages = -(-tokens // page) + 3
    dt = R.TORCH[dtype]
    x = torch.from_numpy(rng.normal(0, 1, size=(tokens, q_heads + 2 * heads, dim)).astype(np.float32)).to(dt)
    if special:  # rows of zeros, of tiny and of large values
        x[0::4] = 0
        x[1::4] *= 2.0**-12
        x[2::4] *= 100.0
    parts = x[:, :q_heads], x[:, q_heads:q_heads + heads], x[:, q_heads + heads:]
    cu = x.cuda()
    dev = [cu[:, :q_heads], cu[:, q_heads:q_heads + heads], cu[:, q_heads + heads:]]
    if not fused:
        dev = [t.contiguous() for t in dev]
    k, ks = R.make_pages(cache, num_pages, heads, page, dim, rng)
    v, vs = R.make_pages(cache, num_pages, heads, page, dim, rng)
    slots = rng.permutation(num_pages * page)[:tokens].astype(np.int64)
    if bad_slots:
        slots[::3] = -1
        slots[1::5] = num_pages * page + np.arange(slots[1::5].size)
        slots[2::7] = -(1 << 40)
    axes = 1 if sections is None else len(sections)
    cs = table_of(200, rot) if rot else None
    pos = rng.integers(0, 200, size=(axes, tokens)).astype(np.int32)
    if bad_positions:
        pos[:, ::4] = -1
        pos[-1, 1::4] = 200
        pos[0, 2::4] = 2**31 - 1
    idx = rng.integers(0, 1 << 30, size=tokens).astype(np.int32)
    w = torch.from_numpy(rng.random((num_pages, heads, page)).astype(np.float32))
    ix = torch.from_numpy(rng.integers(0, 100, size=(num_pages, heads, page)).astype(np.int32))
    d = [t.cuda() if t is not None else None for t in (k, v, ks, vs, w if track else None, ix if track else None)]
    out = nve_kv.kv_append(dev[1], dev[2], d[0], d[1], torch.from_numpy(slots).cuda(), q=dev[0] if with_q else None,
                           positions=torch.from_numpy(pos if axes > 1 else pos[0]).cuda(),
                           cos_sin=None if cs is None else torch.from_numpy(cs).cuda(), sections=sections,
                           interleaved=interleaved, index=torch.from_numpy(idx).cuda() if index else None,
                           k_scale=d[2], v_scale=d[3], weights=d[4], index_pages=d[5])
    torch.cuda.synchronize()
    secs = sections if sections is not None else [rot // 2]
    rq = R.rotate(parts[0], pos, cs, secs, interleaved)
    rk = R.rotate(parts[1], pos, cs, secs, interleaved)
    if with_q:
        assert torch.equal(out.cpu(), torch.from_numpy(rq).to(dt))
    else:
        assert out is None
    there = (slots >= 0) & (slots < num_pages * page)
    p, o = torch.from_numpy(slots[there] // page), torch.from_numpy(slots[there] % page)
    pick = torch.from_numpy(there)
    for name, got, scale, pages, rows in (("k", d[0], d[2], k, rk), ("v", d[1], d[3], v, parts[2].float().numpy())):
        want, wscale = pages.clone(), None if scale is None else (ks if name == "k" else vs).clone()
        if cache == "e4m3":
            codes, sc = R.quantize(rows)
            want.view(torch.uint8)[p, :, o] = codes.view(torch.uint8)[pick]
            wscale[p, :, o] = sc[pick]
            assert torch.equal(scale.cpu(), wscale), name
        else:
            want[p, :, o] = torch.from_numpy(rows).to(dt)[pick]
        # the sign of a zero code is the sign of its value
        assert torch.equal(bits(got.cpu()), bits(want)), name
    if track:
        w[p, :, o] = 0.0
        ix[p, :, o] = torch.from_numpy(idx if index else pos[0])[pick][:, None]
        assert torch.equal(d[4].cpu(), w) and torch.equal(d[5].cpu(), ix)
    return parts, pos, cs, rq


LAYOUTS = [(8, 2, 128, 16, 128, None), (4, 4, 64, 8, 64, None), (6, 3, 96, 64, 64, [12, 10, 10]),
           (20, 1, 80, 16, 80, [20, 20]), (2, 1, 256, 32, 256, [64, 32, 16, 16]), (3, 1, 8, 8, 8, None),
           (5, 5, 72, 16, 34, [17]), (1, 1, 200, 1024, 2, None), (8, 2, 128, 16, 0, None), (3, 3, 40, 8, 24, [0, 12, 0])]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("q_heads,heads,dim,page,rot,sections", LAYOUTS)
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_rows(dtype, cache, q_heads, heads, dim, page, rot, sections, interleaved):
    run(dtype, cache, 37, q_heads, heads, dim, page, rot, sections, interleaved, seed=dim + rot)


@pytest.mark.parametrize("tokens", [1, 2, 3, 63, 64, 65, 1000, 4099])
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_token_counts(dtype, cache, tokens):
    run(dtype, cache, tokens, 4, 2, 64, 16, 64, seed=tokens, fused=True)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_what_is_out_of_range_is_left_alone(dtype, cache, interleaved):
    run(dtype, cache, 50, 4, 2, 64, 16, 48, [12, 12], interleaved, seed=1, bad_slots=True, bad_positions=True)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_zero_tiny_and_large_rows(dtype, cache):
    run(dtype, cache, 41, 4, 2, 64, 16, 64, seed=2, special=True)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_optional_parts(dtype, cache):
    run(dtype, cache, 19, 4, 2, 64, 16, 64, seed=3, index=False)
    run(dtype, cache, 19, 4, 2, 64, 16, 64, seed=4, track=False)
    run(dtype, cache, 19, 4, 2, 64, 16, 64, seed=5, with_q=False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_odd_strides_and_offsets(dtype):
    """Head rows that start at any element, heads and tokens apart by odd distances, heads outermost."""
    from pynve.torch import nve_kv

    rng = np.random.default_rng(6)
    n, dim, dt = 21, 64, R.TORCH[dtype]
    cs = torch.from_numpy(table_of(50, dim)).cuda()
    pos = torch.from_numpy(rng.integers(0, 50, size=n).astype(np.int32)).cuda()
    slots = torch.arange(n).cuda()
    base = torch.from_numpy(rng.normal(0, 1, size=(n, 7, 67)).astype(np.float32)).to(dt).cuda()
    heads_first = torch.from_numpy(rng.normal(0, 1, size=(2, n, 64)).astype(np.float32)).to(dt).cuda()

    def go(q, k, v):
        pages = [torch.zeros((2, 2, 16, dim), dtype=dt, device="cuda") for _ in range(2)]
        out = nve_kv.kv_append(k, v, *pages, slots, q=q, positions=pos, cos_sin=cs)
        return [out] + pages

    q, k, v = base[:, :3, 3:], base[:, 3:5, 1:65], heads_first.transpose(0, 1)
    for a, b in zip(go(q, k, v), go(*(t.contiguous() for t in (q, k, v)))):
        assert torch.equal(a, b)


def test_near_the_rotation_in_64_bits():
    parts, pos, cs, rq = run("f32", "f32", 30, 4, 2, 64, 16, 64, seed=7)
    x, c, s = parts[0].double().numpy(), cs[pos[0], :32].astype(np.float64), cs[pos[0], 32:].astype(np.float64)
    a, b = x[..., :32], x[..., 32:]
    want = np.concatenate([a * c[:, None] - b * s[:, None], b * c[:, None] + a * s[:, None]], -1)
    # two products and a sum, each rounded: 2^-24 of the magnitudes each
    bound = 2.0**-23 * (np.abs(np.concatenate([a * c[:, None], b * c[:, None]], -1)) +
                        np.abs(np.concatenate([b * s[:, None], a * s[:, None]], -1)))
    assert (np.abs(rq - want) <= bound).all()


def test_nan_and_infinity_in_e4m3_rows():
    """A row with a NaN has a NaN scale; the other rows of the call are as ever."""
    from pynve.torch import nve_kv

    k = torch.randn(4, 1, 64, device="cuda").half()
    want_k = k.clone()
    k[1, 0, 7] = float("nan")
    pages = [torch.zeros((1, 1, 16, 64), dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2)]
    scales = [torch.zeros((1, 1, 16), device="cuda") for _ in range(2)]
    nve_kv.kv_append(k, want_k, *pages, torch.arange(4).cuda(), k_scale=scales[0], v_scale=scales[1])
    assert torch.isnan(scales[0][0, 0, 1])
    for i in (0, 2, 3):
        assert torch.equal(bits(pages[0])[0, 0, i], bits(pages[1])[0, 0, i]) and scales[0][0, 0, i] == scales[1][0, 0, i]


def test_no_tokens():
    from pynve.torch import nve_kv

    pages = [torch.zeros((1, 2, 16, 64), dtype=torch.float16, device="cuda") for _ in range(2)]
    e = torch.zeros((0, 2, 64), dtype=torch.float16, device="cuda")
    out = nve_kv.kv_append(e, e, *pages, torch.zeros(0, dtype=torch.int64, device="cuda"), q=e)
    assert out.shape == (0, 2, 64)


def test_refusals():
    from pynve.torch import nve_kv

    def run(**c):
        a = {"k": torch.zeros((3, 2, 64), dtype=torch.float16, device="cuda"),
             "kp": torch.zeros((2, 2, 16, 64), dtype=torch.float16, device="cuda"),
             "slots": torch.arange(3).cuda(), "positions": torch.zeros(3, dtype=torch.int32, device="cuda"),
             "cos_sin": torch.zeros((4, 64), device="cuda")}
        a["v"], a["vp"], a["q"] = torch.zeros_like(a["k"]), torch.zeros_like(a["kp"]), torch.zeros_like(a["k"])
        a.update(c)
        k, v, kp, vp, slots = (a.pop(n) for n in ("k", "v", "kp", "vp", "slots"))
        return nve_kv.kv_append(k, v, kp, vp, slots, **a)

    z = lambda *shape, dtype=torch.float16: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
    run()
    for c in [{"k": z(3, 3, 64)}, {"k": z(2, 2, 64)}, {"v": z(3, 2, 56)}, {"q": z(2, 2, 64)}, {"q": z(3, 64)},
              {"slots": torch.arange(2).cuda()}, {"slots": torch.arange(3)}, {"positions": None},
              {"positions": z(2, 3, dtype=torch.int32)}, {"positions": z(5, 3, dtype=torch.int32), "sections": [32, 0, 0, 0, 0]},
              {"positions": z(2, 3, dtype=torch.int32), "sections": [16, 15]},
              {"positions": z(2, 3, dtype=torch.int32), "sections": [33, -1]}, {"sections": [31]}, {"sections": [16, 16]},
              {"cos_sin": z(4, 66, dtype=torch.float32)}, {"cos_sin": z(4, 63, dtype=torch.float32)},
              {"cos_sin": z(4, 128, dtype=torch.float32)[:, ::2]}, {"index": z(2, dtype=torch.int32)},
              {"weights": z(2, 2, 8, dtype=torch.float32)}, {"kp": z(2, 2, 16, 64).transpose(1, 2)},
              {"k_scale": z(2, 2, 16, dtype=torch.float32)}]:
        with pytest.raises(ValueError):
            run(**c)
    for c in [{"slots": z(3, dtype=torch.int32)}, {"k": z(3, 2, 64, dtype=torch.float32)},
              {"q": z(3, 2, 64, dtype=torch.bfloat16)}, {"positions": torch.arange(3).cuda()},
              {"cos_sin": z(4, 64)}, {"index": torch.arange(3).cuda()}]:
        with pytest.raises(TypeError):
            run(**c)
    with pytest.raises(RuntimeError, match="gradient"):
        run(k=z(3, 2, 64).requires_grad_())
