"""A cache of 4-bit values whole: eviction moves codes and scales, bit for bit, and a run of normed
appends, attention and eviction gives what the steps give one by one."""
import numpy as np
import pytest

import kv4_reference as R4
import kv_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def bits(t):
    return t.view(torch.uint8) if t.dtype not in (torch.float32, torch.int32) else t


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("lengths,budget", [([100, 3, 300, 0, 64, 65], 64), ([5000, 1], 500), ([40000], 100)])
def test_eviction(dim, lengths, budget):
    from pynve.torch import nve_kv

    rng = np.random.default_rng(dim)
    heads, page = 2, 16
    num_pages = sum(-(-n // page) for n in lengths) + 2
    shape = (num_pages, heads, page)
    host = [torch.from_numpy(rng.integers(0, 256, size=(*shape, n)).astype(np.uint8))
            for n in (dim // 2, dim // 2, dim // 32, dim // 32)]
    table = R.tables(lengths, page, num_pages, rng, 1)
    w = np.exp(rng.normal(0, 2, size=shape)).astype(np.float32)
    ix = rng.permutation(w.size).reshape(shape).astype(np.int32)
    host += [torch.from_numpy(w), torch.from_numpy(ix)]
    d = [t.cuda() for t in host]
    (k, ks), (v, vs) = R4.typed(d[0], d[2]), R4.typed(d[1], d[3])
    lens = np.asarray(lengths, np.int32)
    new = nve_kv.kv_evict(k, v, d[4], d[5], torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda(), budget,
                          sinks=2, recent=5, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    moves, want_new = R.evict(w, ix, table, lens, budget, 2, 5, page)
    assert moves and new.cpu().tolist() == want_new
    want = [t.clone() for t in host]
    for h, to, of in moves:
        for a, b in zip(want, host):
            a[to[0], h, to[1]] = b[of[0], h, of[1]]
    for a, b in zip(d, want):
        assert torch.equal(a.cpu(), b)


def state(dim=128):
    from pynve.torch.nve_kv import KVCache

    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    c = KVCache(12, 2, dim, dtype=torch.float4_e2m1fn_x2)
    table = torch.randperm(12, device="cuda", generator=g).int().view(3, 4)
    n = 150
    rows = lambda heads, n: torch.randn(n, heads, dim, device="cuda", generator=g).half()  # noqa: E731
    seq, place = torch.arange(n, device="cuda") % 3, torch.arange(n, device="cuda") // 3
    c.append(rows(2, n), rows(2, n), c.slots(table, seq, place), index=place.int())
    lengths = torch.full((3,), 51, device="cuda", dtype=torch.int32)
    slots = c.slots(table, torch.arange(3, device="cuda"), torch.full((3,), 50, device="cuda"))
    angle = torch.rand(60, dim // 2, device="cuda", generator=g)
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1)
    return c, (rows(8, 3), rows(2, 3), rows(2, 3), slots, table, lengths, lengths - 1, cos_sin,
               torch.rand(dim, device="cuda", generator=g).half())


def step(c, q, k, v, slots, table, lengths, at, cos_sin, norm):
    q = c.append(k, v, slots, q=q, positions=at, cos_sin=cos_sin, q_norm=norm, k_norm=norm)
    out, lse = c.attend(q, table, lengths, return_lse=True)
    return q, out, lse, c.evict(table, lengths, 40, sinks=2, recent=8)


def test_a_step_against_its_parts():
    """Norm, rotation, 4-bit rows, attention in 64 bits and eviction by sorting, in the order a decoder calls them."""
    c, args = state()
    q, k, v, slots, table, lengths, at, cos_sin, norm = args
    before = {n: bits(getattr(c, n)).cpu().clone() for n in ("k", "v", "k_scale", "v_scale", "weights", "index")}
    rq, out, lse, new = step(c, *args)
    torch.cuda.synchronize()
    cs, pos = cos_sin.cpu().numpy(), at.cpu().numpy()
    turn = lambda x: R.rotate(torch.from_numpy(R4.norm(x.cpu(), norm.cpu(), 1e-6)), pos, cs, [64], False)  # noqa: E731
    assert torch.equal(rq.cpu(), torch.from_numpy(turn(q)).half())
    p, o = (slots // 16).cpu(), (slots % 16).cpu()
    for name, rows in (("k", turn(k)), ("v", v.float().cpu().numpy())):
        before[name][p, :, o], before[name + "_scale"][p, :, o] = R4.quantize(rows)
    before["weights"][p, :, o], before["index"][p, :, o] = 0.0, at.cpu()[:, None]
    want = R.attend(rq.cpu(), R4.values64(before["k"], before["k_scale"]), R4.values64(before["v"], before["v_scale"]),
                    table.cpu().numpy(), [51] * 3, 128**-0.5, "f16", "mxfp4")
    assert (np.abs(out.cpu().double().numpy() - want[0]) <= want[3]).all()
    assert (np.abs(lse.cpu().double().numpy() - want[1]) <= want[4]).all()
    # 51 slots are cut to 40: what stays are 40 of the rows that were there, each with its scales
    assert new.cpu().tolist() == [40] * 3
    for s in range(3):
        was = [(int(table[s, t // 16]), t % 16) for t in range(51)]
        for h in range(2):
            old = {tuple(before["k"][a, h, b].tolist() + before["k_scale"][a, h, b].tolist() +
                         before["v"][a, h, b].tolist() + before["v_scale"][a, h, b].tolist()) for a, b in was}
            now = {tuple(x for n in ("k", "k_scale", "v", "v_scale") for x in bits(getattr(c, n))[a, h, b].tolist())
                   for a, b in was[:40]}
            assert len(now) == 40 and now <= old


def test_a_compiled_step():
    a, b = state(), state()
    want = step(a[0], *a[1])
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(b[0], *b[1])
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    for name in ("k", "v", "k_scale", "v_scale", "weights", "index"):
        assert torch.equal(bits(getattr(b[0], name)), bits(getattr(a[0], name))), name


def test_schema_says_what_is_written():
    c, (q, k, v, slots, table, lengths, at, cos_sin, norm) = state()
    d = type(c)(12, 2, 128, dtype=torch.float16)
    torch.library.opcheck(torch.ops.nve_ops.kv_append_norm.default,
                          (k, v, d.k, d.v, slots, q, at, cos_sin, None, False, None, None, None, d.weights, d.index, norm,
                           norm, 1e-6), test_utils=("test_schema", "test_faketensor"))
