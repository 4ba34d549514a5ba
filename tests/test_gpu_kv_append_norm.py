"""New tokens entering the cache with norms of their query and key heads, and rows entering 4-bit pages
(nve_ops::kv_append_norm, kv_append): bit for bit what the definition's steps give (kv4_reference,
kv_reference), over types, layouts, rotations, strides and special rows; what is not written stays."""
import numpy as np
import pytest

import kv4_reference as R4
import kv_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "e4m3"), ("bf16", "e4m3"), ("f16", "mxfp4"),
         ("bf16", "mxfp4")]
MX = [t for t in TYPES if t[1] == "mxfp4"]


def bits(t):
    return t.contiguous().view(torch.uint8)


def same(a, b):
    """Bit for bit, but for what a NaN holds besides."""
    a, b = (t if t.dtype != torch.float8_e4m3fn else t.float() for t in (a, b))
    nan = torch.isnan(b)
    return bool((torch.isnan(a) == nan).all() and torch.equal(bits(a[~nan]), bits(b[~nan])))


def table_of(positions, rot):
    a = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(0, rot, 2) / max(rot, 1))
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


def make_pages(cache, *shape_rng):
    return R4.make_pages(*shape_rng) if cache == "mxfp4" else R.make_pages(cache, *shape_rng)


def run(dtype, cache, tokens, q_heads, heads, dim, page, rot=0, sections=None, interleaved=False, seed=0, fused=False,
        bad=False, norms="qk", eps=1e-6, edit=None):
    from pynve.torch import nve_kv

    rng = np.random.default_rng(seed)
    num_pages = -(-tokens // page) + 3
    dt = R.TORCH[dtype]
    x = torch.from_numpy(rng.normal(0, 1, size=(tokens, q_heads + 2 * heads, dim)).astype(np.float32)).to(dt)
    if edit:
        edit(x)
    parts = x[:, :q_heads], x[:, q_heads:q_heads + heads], x[:, q_heads + heads:]
    cu = x.cuda()
    dev = [cu[:, :q_heads], cu[:, q_heads:q_heads + heads], cu[:, q_heads + heads:]]
    if not fused:
        dev = [t.contiguous() for t in dev]
    k, ks = make_pages(cache, num_pages, heads, page, dim, rng)
    v, vs = make_pages(cache, num_pages, heads, page, dim, rng)
    slots = rng.permutation(num_pages * page)[:tokens].astype(np.int64)
    axes = 1 if sections is None else len(sections)
    cs = table_of(200, rot) if rot else None
    pos = rng.integers(0, 200, size=(axes, tokens)).astype(np.int32)
    if bad:
        slots[::3] = -1
        slots[1::5] = num_pages * page + np.arange(slots[1::5].size)
        pos[:, ::4] = -1
        pos[-1, 1::4] = 200
    weight = {n: torch.from_numpy(np.exp(rng.normal(0, 0.5, size=dim)).astype(np.float32)).to(dt) for n in "qk"}
    w = torch.from_numpy(rng.random((num_pages, heads, page)).astype(np.float32))
    ix = torch.from_numpy(rng.integers(0, 100, size=(num_pages, heads, page)).astype(np.int32))
    d = [t.cuda() if t is not None else None for t in (k, v, ks, vs, w, ix)]
    mx = cache == "mxfp4"
    typed = [*(t.view(torch.float4_e2m1fn_x2) for t in d[:2]),
             *(t.view(torch.float8_e8m0fnu) for t in d[2:4])] if mx else d[:4]
    out = nve_kv.kv_append(dev[1], dev[2], typed[0], typed[1], torch.from_numpy(slots).cuda(), q=dev[0],
                           positions=torch.from_numpy(pos if axes > 1 else pos[0]).cuda(),
                           cos_sin=None if cs is None else torch.from_numpy(cs).cuda(), sections=sections,
                           interleaved=interleaved, k_scale=typed[2], v_scale=typed[3], weights=d[4], index_pages=d[5],
                           q_norm=weight["q"].cuda() if "q" in norms else None,
                           k_norm=weight["k"].cuda() if "k" in norms else None, eps=eps)
    torch.cuda.synchronize()
    secs = sections if sections is not None else [rot // 2]
    rows = [R.rotate(torch.from_numpy(R4.norm(t, weight[n] if n in norms else None, eps)), pos, cs, secs, interleaved)
            for t, n in zip(parts, "qk")] + [parts[2].float().numpy()]
    assert same(out.cpu(), torch.from_numpy(rows[0]).to(dt))
    there = (slots >= 0) & (slots < num_pages * page)
    p, o, pick = torch.from_numpy(slots[there] // page), torch.from_numpy(slots[there] % page), torch.from_numpy(there)
    for name, got, scale, old, old_scale, r in (("k", d[0], d[2], k, ks, rows[1]), ("v", d[1], d[3], v, vs, rows[2])):
        want, wscale = old.clone(), None if scale is None else old_scale.clone()
        if mx:
            codes, sc = R4.quantize(r)
            want[p, :, o], wscale[p, :, o] = codes[pick], sc[pick]
            nans = (wscale == 255).repeat_interleave(16, -1)  # codes under a NaN scale say nothing
            assert torch.equal(scale.cpu(), wscale), name
            assert torch.equal(got.cpu()[~nans], want[~nans]), name
            continue
        if cache == "e4m3":
            codes, sc = R.quantize(r)
            want.view(torch.uint8)[p, :, o] = codes.view(torch.uint8)[pick]
            wscale[p, :, o] = sc[pick]
            assert torch.equal(scale.cpu(), wscale), name
        else:
            want[p, :, o] = torch.from_numpy(r).to(dt)[pick]
        assert same(got.cpu(), want), name
    w[p, :, o] = 0.0
    ix[p, :, o] = torch.from_numpy(pos[0])[pick][:, None]
    assert torch.equal(d[4].cpu(), w) and torch.equal(d[5].cpu(), ix)
    return parts, weight, pos, cs, rows


LAYOUTS = [(8, 2, 128, 16, 128, None), (4, 4, 64, 8, 64, None), (6, 3, 96, 64, 64, [12, 10, 10]),
           (20, 1, 160, 16, 160, [40, 40]), (2, 1, 256, 32, 256, [64, 32, 32]), (5, 5, 192, 16, 34, [17]),
           (8, 2, 128, 16, 0, None), (3, 3, 32, 8, 32, None), (3, 1, 64, 1024, 32, [0, 16, 0]), (2, 2, 224, 8, 128, None)]
ODD = [(3, 1, 8, 8, 8, None), (5, 5, 72, 16, 34, [17]), (1, 1, 200, 32, 2, None), (3, 3, 40, 8, 24, [0, 12, 0]),
       (20, 1, 80, 16, 80, [20, 20])]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_rows(dtype, cache, layout, interleaved):
    run(dtype, cache, 37, *layout, interleaved, seed=layout[2] + layout[4])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ODD)
@pytest.mark.parametrize("dtype,cache", TYPES[:5])
def test_odd_widths(dtype, cache, layout, interleaved):
    run(dtype, cache, 37, *layout, interleaved, seed=layout[2] + layout[4])


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype,cache", MX)
def test_4_bit_rows_without_a_norm(dtype, cache, layout):
    run(dtype, cache, 37, *layout, False, seed=layout[2] + layout[4], norms="")


@pytest.mark.parametrize("tokens", [1, 2, 3, 63, 64, 65, 1000, 4099])
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_token_counts(dtype, cache, tokens):
    run(dtype, cache, tokens, 4, 2, 64, 16, 64, seed=tokens, fused=True)


@pytest.mark.parametrize("rot", [128, 32])
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_one_norm_alone(dtype, cache, rot):
    run(dtype, cache, 21, 4, 2, 128, 16, rot, seed=1, norms="q")
    run(dtype, cache, 21, 4, 2, 128, 16, rot, seed=2, norms="k")


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_what_is_out_of_range_is_left_alone(dtype, cache, interleaved):
    run(dtype, cache, 50, 4, 2, 64, 16, 64, [20, 12], interleaved, seed=1, bad=True)
    run(dtype, cache, 50, 4, 2, 96, 16, 48, [12, 12], interleaved, seed=1, bad=True)


@pytest.mark.parametrize("eps", [0.0, 1e-12, 1e-5, 3.0])
@pytest.mark.parametrize("norms", ["", "qk"])
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_zero_tiny_and_large_rows(dtype, cache, norms, eps):
    def edit(x):
        x[0::5] = 0
        x[1::5] *= 2.0**-12
        x[2::5] *= 100.0
        x[3::5, :, ::7] *= 300.0

    if eps == 0.0 and norms and cache == "e4m3":
        return  # a row of zeros is NaN then, and so is its scale
    run(dtype, cache, 41, 4, 2, 64, 16, 64, seed=2, edit=edit, norms=norms, eps=eps)


@pytest.mark.parametrize("rot", [64, 24])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_zero_rows_without_eps_in_8_bits(dtype, rot):
    """A row of zeros has no norm where eps is 0: NaN, with a NaN for its scale.  The rows beside it are as ever."""
    from pynve.torch import nve_kv

    rng = np.random.default_rng(10)
    dt, n = R.TORCH[dtype], 23
    q, k, v = (torch.from_numpy(rng.normal(0, 1, size=(n, h, 64)).astype(np.float32)).to(dt) for h in (4, 2, 2))
    for x in (q, k, v):
        x[::3] = 0
    k[1, 0] = 0
    weight = {x: torch.from_numpy(np.exp(rng.normal(0, 0.5, size=64)).astype(np.float32)).to(dt) for x in "qk"}
    cs, pos = table_of(50, rot), rng.integers(0, 50, size=(1, n)).astype(np.int32)
    cache = nve_kv.KVCache(3, 2, 64, dtype=torch.float8_e4m3fn)
    out = cache.append(k.cuda(), v.cuda(), torch.arange(n).cuda(), q=q.cuda(), positions=torch.from_numpy(pos[0]).cuda(),
                       cos_sin=torch.from_numpy(cs).cuda(), q_norm=weight["q"].cuda(), k_norm=weight["k"].cuda(), eps=0.0)
    rows = [R.rotate(torch.from_numpy(R4.norm(x, w, 0.0)), pos, cs, [rot // 2], False)
            for x, w in ((q, weight["q"]), (k, weight["k"]))] + [v.float().numpy()]
    assert same(out.cpu(), torch.from_numpy(rows[0]).to(dt))
    at = np.arange(n)
    for pages, scales, r in ((cache.k, cache.k_scale, rows[1]), (cache.v, cache.v_scale, rows[2])):
        got, scale = pages.cpu()[at // 16, :, at % 16].float(), scales.cpu()[at // 16, :, at % 16]
        none = torch.from_numpy(np.isnan(r).any(-1))
        codes, want = R.quantize(np.nan_to_num(r))
        assert torch.equal(torch.isnan(scale), none) and torch.isnan(got[none]).all()
        assert torch.equal(scale[~none], want[~none]) and torch.equal(got[~none], codes[~none].float())
    assert torch.isnan(cache.k_scale.cpu()[0, :, 0]).all() and not torch.isnan(cache.v_scale).any()


@pytest.mark.parametrize("dtype,cache", MX)
@pytest.mark.parametrize("rot", [0, 32, 64])
def test_values_on_the_borders_of_codes_and_scales(dtype, cache, rot):
    """Ties between codes, magnitudes of exactly 7 times a power of two and next to it, the least and largest values."""
    def edit(x):
        flat = x.reshape(-1, 64)
        ties = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7])
        for i in range(flat.shape[0]):
            row = torch.cat([ties, -ties, ties.flip(0) * 0.5, ties * 0.125])
            flat[i] = (row * 2.0 ** (i % 24 - 14)).to(x.dtype)
            if i % 3 == 1:
                flat[i, 15] = torch.nextafter(flat[i, 15], torch.tensor(1e4).to(x.dtype))
            if i % 7 == 2:
                flat[i, 40] = torch.finfo(x.dtype).max
            if i % 7 == 3:
                flat[i] = 0.0
                flat[i, 3] = torch.finfo(x.dtype).tiny

    run(dtype, cache, 48, 2, 2, 64, 16, 0, seed=9, norms="", edit=edit)
    if rot:
        run(dtype, cache, 48, 2, 2, 64, 16, rot, seed=9, norms="", edit=edit)


@pytest.mark.parametrize("dtype,cache", MX)
@pytest.mark.parametrize("rot", [64, 32])
def test_nan_and_infinity_in_4_bit_rows(dtype, cache, rot):
    """32 values with a NaN or an infinity have the scale NaN, the others are as ever."""
    def edit(x):
        x[1, :, 40] = float("nan")
        x[2, :, 3] = float("inf")
        x[3, :, 33] = -float("inf")

    run(dtype, cache, 9, 2, 2, 64, 16, 0, seed=4, norms="", edit=edit)
    run(dtype, cache, 9, 2, 2, 96, 16, rot, seed=4, norms="", edit=edit)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mx", [False, True])
def test_odd_strides_and_offsets(dtype, mx):
    """Head rows that start at any element, heads and tokens apart by odd distances, heads outermost."""
    from pynve.torch import nve_kv

    if mx and dtype == "f32":
        return
    rng = np.random.default_rng(6)
    n, dim, dt = 21, 64, R.TORCH[dtype]
    cs = torch.from_numpy(table_of(50, dim)).cuda()
    pos = torch.from_numpy(rng.integers(0, 50, size=n).astype(np.int32)).cuda()
    slots = torch.arange(n).cuda()
    base = torch.from_numpy(rng.normal(0, 1, size=(n, 7, 67)).astype(np.float32)).to(dt).cuda()
    heads_first = torch.from_numpy(rng.normal(0, 1, size=(2, n, 64)).astype(np.float32)).to(dt).cuda()
    weight = torch.rand(dim + 1, device="cuda").to(dt)[1:]

    def go(q, k, v):
        cache = nve_kv.KVCache(2, 2, dim, dtype=torch.float4_e2m1fn_x2 if mx else dt)
        out = cache.append(k, v, slots, q=q, positions=pos, cos_sin=cs, q_norm=weight, k_norm=weight)
        return [out] + [bits(t) for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]

    q, k, v = base[:, :3, 3:], base[:, 3:5, 1:65], heads_first.transpose(0, 1)
    for a, b in zip(go(q, k, v), go(*(t.contiguous() for t in (q, k, v)))):
        assert torch.equal(a, b)


def test_near_the_norm_and_rotation_in_64_bits():
    parts, weight, pos, cs, rows = run("f32", "f32", 30, 4, 2, 64, 16, 64, seed=7)
    c, s = cs[pos[0], :32].astype(np.float64)[:, None], cs[pos[0], 32:].astype(np.float64)[:, None]
    x = parts[0].double().numpy()
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * weight["q"].double().numpy()
    a, b = x[..., :32], x[..., 32:]
    want = np.concatenate([a * c - b * s, b * c + a * s], -1)
    # r, two products of the norm, two of the rotation and a sum, each rounded: 2^-24 of the magnitudes each
    size = np.concatenate([np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)], -1)
    assert (np.abs(rows[0] - want) <= 5.01 * 2.0**-24 * size).all()


def test_graph_replays():
    from pynve.torch import nve_kv

    cache, other = (nve_kv.KVCache(4, 2, 128, dtype=torch.float4_e2m1fn_x2) for _ in range(2))
    q, k, v = (torch.randn(5, h, 128, device="cuda").half() for h in (8, 2, 2))
    slots = torch.arange(5).cuda()
    w = torch.rand(128, device="cuda").half()
    cache.append(k, v, slots, q=q, q_norm=w, k_norm=w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.append(k, v, slots, q=q, q_norm=w, k_norm=w)
    for i in range(4):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device="cuda"))
        slots.copy_(torch.randperm(64)[:5])
        graph.replay()
        torch.cuda.synchronize()
        want = other.append(k, v, slots, q=q, q_norm=w, k_norm=w)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for name in ("k", "v", "k_scale", "v_scale"):
            a, b = bits(getattr(cache, name)), bits(getattr(other, name))
            at = (slots // 16, slice(None), slots % 16)
            assert torch.equal(a[at], b[at]), name


def test_refusals():
    from pynve.torch import nve_kv

    z = lambda *shape, dtype=torch.float16: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731

    def run(**c):
        cache = nve_kv.KVCache(2, 2, 64, dtype=c.pop("dtype", torch.float4_e2m1fn_x2))
        a = {"k": z(3, 2, 64), "v": z(3, 2, 64), "q": z(3, 4, 64), "q_norm": z(64), "k_norm": z(64), "eps": 1e-6, **c}
        return cache.append(a.pop("k"), a.pop("v"), torch.arange(3).cuda(), **a)

    run()
    run(dtype=torch.float16)
    for c in [{"q_norm": z(63)}, {"k_norm": z(64, 1)}, {"k_norm": z(128)[::2]}, {"q_norm": z(64).cpu()}, {"q": None},
              {"eps": -1.0}, {"eps": float("nan")}, {"eps": float("inf")}, {"k": z(3, 2, 32)},
              {"k": z(3, 2, 64, dtype=torch.float32), "v": z(3, 2, 64, dtype=torch.float32),
               "q": z(3, 4, 64, dtype=torch.float32), "q_norm": None, "k_norm": None}]:
        with pytest.raises(ValueError):
            run(**c)
    for c in [{"q_norm": z(64, dtype=torch.float32)}, {"k_norm": z(64, dtype=torch.bfloat16)}]:
        with pytest.raises(TypeError):
            run(**c)
    for name in ("q_norm", "k_norm"):
        with pytest.raises(RuntimeError, match=f"{name} asks for a gradient"):
            run(**{name: z(64).requires_grad_()})
        with torch.no_grad():
            run(**{name: z(64).requires_grad_()})
    with pytest.raises(ValueError):
        nve_kv.KVCache(2, 2, 48, dtype=torch.float4_e2m1fn_x2)
