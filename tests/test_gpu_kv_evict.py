"""Eviction from the paged key-value cache (nve_ops::kv_evict) against sorting:
which slots go, which rows move where, and that nothing else changes, bit for
bit, over ties, NaN and infinite weights, protected slots, lengths and budgets
of every kind."""
import numpy as np
import pytest

import kv_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def bits(t):
    return t.contiguous().view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def run(lengths, budget, heads=2, dim=16, page=16, cache="f16", sinks=0, recent=0, seed=0, weights=None, index=None,
        edit=None, extra=1):
    from pynve.torch import nve_kv

    rng = np.random.default_rng(seed)
    num_pages = sum(-(-max(n, 0) // page) for n in lengths) + 2
    k, ks = R.make_pages(cache, num_pages, heads, page, dim, rng)
    v, vs = R.make_pages(cache, num_pages, heads, page, dim, rng)
    table = R.tables([max(n, 0) for n in lengths], page, num_pages, rng, extra)
    shape = (num_pages, heads, page)
    w = np.exp(rng.normal(0, 2, size=shape)).astype(np.float32) if weights is None else weights(rng, shape)
    ix = np.zeros(shape, np.int32)
    for s, n in enumerate(lengths):
        n = max(n, 0)
        for h in range(heads):
            place = rng.permutation(n) if index is None else index(rng, n)
            t, p, o = R.slots_of(table[s], n, page, num_pages)
            ix[p, h, o] = place
    lens = np.asarray(lengths, np.int32)
    if edit:
        edit(table, lens, w, ix)
    host = [k, v, ks, vs, torch.from_numpy(w), torch.from_numpy(ix)]
    dev = [None if t is None else t.cuda() for t in host]
    new = nve_kv.kv_evict(dev[0], dev[1], dev[4], dev[5], torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda(),
                          budget, sinks=sinks, recent=recent, k_scale=dev[2], v_scale=dev[3])
    torch.cuda.synchronize()
    moves, want_new = R.evict(w, ix, table, lens, budget, sinks, recent, page)
    assert new.cpu().tolist() == want_new and new.dtype == torch.int32
    before = [None if t is None else bits(t).clone() for t in host]
    want = [None if t is None else t.clone() for t in before]
    for h, to, of in moves:
        for a, b in zip(want, before):
            if a is not None:
                a[to[0], h, to[1]] = b[of[0], h, of[1]]
    for name, a, b in zip(("k", "v", "k_scale", "v_scale", "weights", "index"), dev, want):
        if a is not None:
            got = bits(a.cpu())
            if name == "weights":
                got, b = got.view(torch.int32), b.view(torch.int32)
            assert torch.equal(got, b), name
    return moves


@pytest.mark.parametrize("cache,dim", [("f32", 64), ("f16", 8), ("bf16", 136), ("e4m3", 8), ("e4m3", 96), ("f16", 256)])
@pytest.mark.parametrize("page", [8, 64])
def test_types(cache, dim, page):
    assert run([100, 3, 300, 0, 64, 65], 64, 3, dim, page, cache, sinks=2, recent=5, seed=dim)


@pytest.mark.parametrize("budget", [0, 1, 2, 31, 32, 33, 63, 64, 65, 500, 1 << 62])
def test_budgets(budget):
    run([0, 1, 2, 31, 32, 33, 64, 65, 200, 499, 500, 501], budget, seed=1, recent=4, sinks=1)


@pytest.mark.parametrize("lengths,budget", [([1023, 1024, 1025, 1500], 1024), ([2047, 2048, 2049, 5000], 1000),
                                            ([40000], 100), ([40000], 39990), ([33000, 20], 16000)])
def test_long_sequences(lengths, budget):
    run(lengths, budget, heads=1, seed=2, recent=20, sinks=4)


def test_many_sequences():
    rng = np.random.default_rng(3)
    run([int(n) for n in rng.integers(0, 60, size=400)], 20, heads=3, dim=8, page=8, seed=3, recent=3)


@pytest.mark.parametrize("levels", [1, 2, 5])
@pytest.mark.parametrize("recent", [0, 7, 2000])
def test_equal_weights_go_in_slot_order(levels, recent):
    run([1200, 70, 33], 40, seed=4, recent=recent,
        weights=lambda rng, s: rng.integers(0, levels, size=s).astype(np.float32) - 1.0)


def test_zeros_of_both_signs_are_equal():
    run([300, 50], 30, seed=5, weights=lambda rng, s: np.where(rng.random(s) < 0.5, np.float32(-0.0), np.float32(0.0)))


def test_nan_and_infinite_weights():
    def w(rng, s):
        x = rng.normal(0, 1, size=s).astype(np.float32)
        x[rng.random(s) < 0.2] = np.nan
        x[rng.random(s) < 0.1] = -np.nan
        x[rng.random(s) < 0.2] = np.inf
        x[rng.random(s) < 0.2] = -np.inf
        return x

    for budget in (5, 60, 150, 290):
        run([300, 299, 61], budget, seed=6, weights=w, recent=10)


@pytest.mark.parametrize("length", [20, 300, 1024, 1500, 6000, 20000, 40000])
@pytest.mark.parametrize("nans", ["one a page", "some", "all"])
@pytest.mark.parametrize("shuffled", [False, True])
def test_a_budget_of_the_protected_slots_drops_every_other_one(length, nans, shuffled):
    """As many unprotected slots as have to go, NaN weights among them: no protected slot goes with them
    (every kernel variant: 1,024, 4,096, 16,384, 32,768 slots and more)."""
    budget = 5 if length == 20 else 40
    sinks = 2 if length == 20 else 8

    def w(rng, s):
        x = rng.normal(1, 1, size=s).astype(np.float32)
        if nans == "one a page":
            x[:, :, s[2] - 6] = np.nan
        elif nans == "some":
            x[rng.random(s) < 0.1] = np.nan
        else:
            x[:] = np.nan
        return x

    index = None if shuffled else lambda rng, n: np.arange(n)
    run([length, length - 1, budget + 1, budget], budget, heads=1, dim=8, page=16, sinks=sinks, recent=budget - sinks,
        seed=20 + length, weights=w, index=index, extra=0)


def test_negative_tiny_and_close_weights():
    run([900], 300, seed=7, weights=lambda rng, s: (rng.integers(-3, 4, size=s) * np.float32(1e-45)).astype(np.float32))
    run([900], 300, seed=8, weights=lambda rng, s: np.nextafter(np.float32(1), np.float32(2)) *
        (1 + rng.integers(0, 3, size=s) * np.float32(2.0**-23)).astype(np.float32))


@pytest.mark.parametrize("sinks,recent", [(1000, 0), (0, 1 << 62), (10, 100), (0, 1), (50, 0)])
def test_protected_slots(sinks, recent):
    """More protected slots than the budget: the lightest protected ones go too."""
    run([200, 64, 30], 40, seed=9, sinks=sinks, recent=recent)


def test_indices_of_any_kind():
    """Equal, negative and largest indices: places are compared as numbers, without wrapping."""
    for seed, pick in enumerate([lambda r, n: np.zeros(n), lambda r, n: r.integers(-(2**31), 2**31, size=n),
                                 lambda r, n: np.full(n, 2**31 - 1)]):
        run([300, 40], 30, seed=10 + seed, sinks=3, recent=50, index=lambda r, n: pick(r, n).astype(np.int32))


def test_absent_pages():
    def edit(table, lens, w, ix):
        table[0, 2], table[0, 9], table[1, 0] = -1, 1 << 30, w.shape[0]

    run([300, 100], 64, seed=13, edit=edit, recent=10)


def test_length_bounds():
    def edit(table, lens, w, ix):
        lens[0], lens[1] = 2**31 - 1, -4

    run([320, 32, 64], 50, seed=14, edit=edit, extra=0)


def test_the_evicted_sequence_attends_to_what_is_kept():
    """Append, attend with accumulation, evict, attend: the output over the kept slots, in 64 bits."""
    from pynve.torch.nve_kv import KVCache

    rng = np.random.default_rng(15)
    heads, dim, n, budget = 2, 64, 100, 40
    c = KVCache(10, heads, dim, dtype=torch.float32)
    table = torch.tensor([[7, 2, 9, 4, 0, 1, 3]], dtype=torch.int32, device="cuda")
    k, v = (torch.from_numpy(rng.normal(0, 1, (n, heads, dim)).astype(np.float32)).cuda() for _ in range(2))
    place = torch.arange(n, device="cuda")
    c.append(k, v, c.slots(table, torch.zeros_like(place), place), index=place.int())
    q = torch.from_numpy(rng.normal(0, 2, (1, 2 * heads, dim)).astype(np.float32)).cuda()
    length = torch.tensor([n], dtype=torch.int32, device="cuda")
    c.attend(q, table, length)
    p = torch.softmax(torch.einsum("hd,thd->ht", q[0].double().cpu(), k.double().cpu().repeat_interleave(2, 1)) / 8, -1)
    w = p.view(heads, 2, n).sum(1)
    length = c.evict(table, length, budget, recent=8, sinks=2)
    assert length.item() == budget
    got = c.attend(q, table, length, accumulate=False)[0].cpu()
    for h in range(heads):
        kept = set(range(2)) | set(range(n - 8, n))
        order = sorted((t for t in range(n) if t not in kept), key=lambda t: -w[h, t])
        kept = sorted(kept | set(order[:budget - len(kept)]))
        for g in range(2):
            x = (k[kept, h].double().cpu() @ q[0, 2 * h + g].double().cpu()) / 8
            want = torch.softmax(x, -1) @ v[kept, h].double().cpu()
            assert (got[2 * h + g].double() - want).abs().max() < 1e-5


def test_more_heads_than_a_launch_has_workgroups():
    """65,535 sequences of 257 heads, more than 2^32 threads of the kernel that moves rows; only the
    first and the last are over the budget, and come out as they do by themselves."""
    from pynve.torch import nve_kv

    seqs, heads, page, dim, per = 65535, 257, 8, 8, 17
    g = torch.Generator(device="cuda")
    g.manual_seed(17)
    shape = (2 * per, heads, page)
    first = [torch.randn((*shape, dim), device="cuda", generator=g).half() for _ in range(2)]
    first += [torch.rand(shape, device="cuda", generator=g)]
    first += [torch.arange(per * page, device="cuda", dtype=torch.int32).view(per, 1, page).repeat(2, heads, 1)]
    small = torch.arange(2 * per, device="cuda", dtype=torch.int32).view(2, per)
    table = torch.full((seqs, per), -1, device="cuda", dtype=torch.int32)
    lengths = torch.zeros(seqs, device="cuda", dtype=torch.int32)
    table[0], table[-1] = small[0], small[1]
    lengths[0] = lengths[-1] = per * page
    got, want = [t.clone() for t in first], [t.clone() for t in first]
    new = nve_kv.kv_evict(*got, table, lengths, 65, recent=5)
    nve_kv.kv_evict(*want, small, torch.full((2,), per * page, device="cuda", dtype=torch.int32), 65, recent=5)
    torch.cuda.synchronize()
    assert new[0] == new[-1] == 65 and new.sum() == 130
    assert not torch.equal(want[0], first[0])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graph_replays():
    from pynve.torch import nve_kv

    rng = np.random.default_rng(16)
    shape, lens = (60, 2, 16), [500, 300]
    k = torch.randn((*shape, 16), device="cuda")
    v = torch.randn_like(k)
    w = torch.zeros(shape, device="cuda")
    ix = torch.zeros(shape, dtype=torch.int32, device="cuda")
    table = torch.from_numpy(R.tables(lens, 16, 60, rng)).cuda()
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    args = lambda: (k, v, w, ix, table, length, 100)  # noqa: E731
    nve_kv.kv_evict(*args())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new = nve_kv.kv_evict(*args())
    for i in range(4):
        w.copy_(torch.rand(shape, device="cuda"))
        length.copy_(torch.tensor([500 - 120 * i, 300 - i], dtype=torch.int32))
        state = [t.clone() for t in (k, v, w, ix)]
        graph.replay()
        torch.cuda.synchronize()
        want = nve_kv.kv_evict(*state, table, length, 100)
        torch.cuda.synchronize()
        assert torch.equal(new, want)
        assert all(torch.equal(a, b) for a, b in zip((k, v, w, ix), state))


def test_refusals():
    from pynve.torch import nve_kv
    from pynve.torch.nve_kv import KVCache

    def run(**c):
        a = {"k": torch.zeros((2, 2, 16, 64), dtype=torch.float16, device="cuda"),
             "w": torch.zeros((2, 2, 16), device="cuda"), "i": torch.zeros((2, 2, 16), dtype=torch.int32, device="cuda"),
             "t": torch.zeros((1, 2), dtype=torch.int32, device="cuda"),
             "n": torch.full((1,), 20, dtype=torch.int32, device="cuda"), "budget": 8}
        a["v"] = torch.zeros_like(a["k"])
        a.update(c)
        args = [a.pop(n) for n in ("k", "v", "w", "i", "t", "n", "budget")]
        return nve_kv.kv_evict(*args, **a)

    run()
    for c in [{"budget": -1}, {"sinks": -1}, {"recent": -1}, {"n": torch.zeros(2, dtype=torch.int32, device="cuda")},
              {"t": torch.zeros(2, dtype=torch.int32, device="cuda")}, {"w": torch.zeros((2, 2, 8), device="cuda")},
              {"w": torch.zeros((2, 2, 16))}, {"k_scale": torch.zeros((2, 2, 16), device="cuda")}]:
        with pytest.raises(ValueError):
            run(**c)
    for c in [{"w": torch.zeros((2, 2, 16), device="cuda").half()}, {"i": torch.zeros((2, 2, 16), device="cuda").long()},
              {"t": torch.zeros((1, 2), device="cuda").long()}]:
        with pytest.raises(TypeError):
            run(**c)
    c = KVCache(2, 2, 64, track_weights=False)
    with pytest.raises(ValueError):
        c.evict(torch.zeros((1, 2), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), 8)
