"""Token sampling (nve_ops::sample_tokens) against sorting and running sums in 64 bits, token for token:
types, vocabularies from one token on, every limit and their mixtures, ties, masks, infinities and NaN,
extreme temperatures and random numbers, strides, streams and graphs."""
import math

import numpy as np
import pytest

import sample_reference as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LIMITS = [{}, {"temperature": 0.7}, {"top_k": 1}, {"top_k": 5}, {"top_k": 50, "temperature": 0.8}, {"top_p": 0.9},
          {"top_p": 0.3, "temperature": 1.5}, {"min_p": 0.05}, {"top_k": 40, "top_p": 0.95, "min_p": 0.02},
          {"temperature": 0.0}, {"top_k": 700, "top_p": 0.999}, {"top_p": 0.9999}, {"top_p": 0.0}, {"min_p": 1.0},
          {"top_k": 3000, "temperature": 2.0}]


def logits_of(rng, rows, vocab, spread=2.0, dtype="f32"):
    x = rng.normal(0, spread, size=(rows, vocab))
    few = max(1, vocab // 50)
    for r in range(rows):  # what a context suggests
        at = rng.integers(0, vocab, size=few)
        x[r, at] += rng.exponential(spread * 3 * rng.random(), size=few)
    return torch.from_numpy(x.astype(np.float32)).to(TYPES[dtype])


def cuda(x):
    return (torch.from_numpy(x) if isinstance(x, np.ndarray) else x).cuda()


def check(x, u, **limits):
    from pynve.torch.nve_sample import sample_tokens

    u = np.asarray(u, np.float32)
    dev = {n: cuda(np.asarray(v, np.int32 if n == "top_k" else np.float32)) if np.ndim(v) else v for n, v in limits.items()}
    got = sample_tokens(cuda(x), cuda(u), **dev)
    assert got.dtype == torch.int64 and got.shape == (x.shape[0],)
    got = got.cpu().numpy()
    want = R.sample(x.float().numpy(), u, **limits)
    bad = np.flatnonzero(got != want)
    assert bad.size == 0, f"{bad.size} rows, first {bad[0]}: {got[bad[0]]} for {want[bad[0]]}"
    return got


@pytest.mark.parametrize("limits", LIMITS)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [1000, 32003])
def test_limits(dtype, vocab, limits):
    rng = np.random.default_rng(vocab)
    check(logits_of(rng, 24, vocab, dtype=dtype), rng.random(24), **limits)


@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 63, 64, 65, 127, 255, 257, 511, 513, 1023, 1024, 1025, 2047, 2049, 4095, 4097,
                                   8191, 8193, 16385, 50257, 65536, 131072, 131073, 262147])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_vocabularies(dtype, vocab):
    rng = np.random.default_rng(vocab)
    n = 12 if vocab < 60000 else 5
    x = logits_of(rng, n, vocab, dtype=dtype)
    for limits in ({}, {"top_k": 20, "top_p": 0.9}, {"top_p": 0.8}, {"min_p": 0.1}):
        check(x, rng.random(n), **limits)


@pytest.mark.parametrize("vocab", [524287, 524288, 524289, 1000003])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_the_largest_vocabularies(dtype, vocab):
    rng = np.random.default_rng(vocab)
    x = logits_of(rng, 2, vocab, dtype=dtype)
    for limits in ({}, {"top_k": 20, "top_p": 0.9}, {"top_p": 0.8}, {"min_p": 0.1}, {"temperature": 0.0}):
        check(x, rng.random(2), **limits)


@pytest.mark.parametrize("limits", [{}, {"top_k": 9}, {"top_p": 0.9}, {"top_p": 0.99, "min_p": 0.001}])
@pytest.mark.parametrize("rows, vocab", [(2049, 2500), (4100, 40), (300, 140000)])
def test_more_rows_than_a_launch(rows, vocab, limits):
    """Past 2,048 rows, or 256 of a large vocabulary, the workspace is used again."""
    rng = np.random.default_rng(rows)
    check(logits_of(rng, rows, vocab, spread=0.5 if rows % 100 else 2.0, dtype="bf16"), rng.random(rows), **limits)


@pytest.mark.parametrize("limits", [{"top_p": 0.9}, {"top_p": 0.97, "min_p": 0.05}, {"min_p": 0.3}])
@pytest.mark.parametrize("rows", [257, 400, 700, 1100])
def test_many_wide_rows(rows, limits):
    """Rows with wide nuclei by fewer and fewer slices."""
    rng = np.random.default_rng(rows)
    for dtype in ("f32", "bf16"):
        x = torch.from_numpy(rng.normal(0, 0.7, size=(rows, 16387)).astype(np.float32)).to(TYPES[dtype])
        check(x, rng.random(rows), **limits)


@pytest.mark.parametrize("rows", [1, 2, 7, 64, 300, 1025])
def test_every_row_has_limits_of_its_own(rows):
    rng = np.random.default_rng(rows)
    vocab = 5003
    x = logits_of(rng, rows, vocab)
    on = lambda v, off: np.where(rng.random(rows) < 0.5, v, off)  # noqa: E731
    check(x, rng.random(rows), temperature=on(rng.uniform(0.2, 2, rows), 1.0) * (rng.random(rows) > 0.1),
          top_k=on(np.exp(rng.uniform(0, 8, rows)).astype(int), 0), top_p=on(rng.uniform(0.01, 1.1, rows), 1.0),
          min_p=on(rng.uniform(0, 0.5, rows), 0.0))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("levels", [1, 2, 3, 10])
def test_equal_logits_go_by_their_index(dtype, levels):
    """Few distinct values: the border of every limit lies among equals."""
    rng = np.random.default_rng(levels)
    for vocab in (7, 1000, 20001):
        x = torch.from_numpy(rng.integers(0, levels, size=(16, vocab)).astype(np.float32)).to(TYPES[dtype])
        for limits in ({}, {"top_k": 3}, {"top_k": vocab // 2}, {"top_p": 0.5}, {"top_p": 0.3, "top_k": vocab - 1},
                       {"min_p": 0.9}, {"top_p": 0.75, "min_p": 0.5}):
            check(x, rng.random(16), **limits)
            check(x, np.arange(16) / 16, **limits)  # on the borders of the shares


@pytest.mark.parametrize("k", [900, 1500, 1999, 2048, 2049])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [5003, 32003, 70001])
def test_many_of_top_k(vocab, dtype, k):
    """As many as the groups whose maxima they are looked for by."""
    rng = np.random.default_rng(vocab + k)
    x = logits_of(rng, 8, vocab, dtype=dtype)
    x[4:, ::2] = -math.inf
    for limits in ({}, {"top_p": 0.97}, {"min_p": 1e-4}):
        check(x, rng.random(8), top_k=k, **limits)


@pytest.mark.parametrize("spread", [0.01, 0.3, 1.0])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_flat_rows_have_wide_nuclei(dtype, spread):
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.normal(0, spread, size=(8, 40001)).astype(np.float32)).to(TYPES[dtype])
    for limits in ({"top_p": 0.5}, {"top_p": 0.9, "top_k": 30000}, {"top_k": 20000}, {"top_p": 0.99, "min_p": 0.3},
                   {"min_p": 0.2}):
        check(x, rng.random(8), **limits)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_masked_rows(dtype):
    """Minus infinity and NaN where a token is not allowed, down to one allowed token and to none."""
    rng = np.random.default_rng(6)
    for vocab in (50, 9001):
        x = logits_of(rng, 20, vocab, dtype=dtype)
        for r in range(20):
            n = [0, 1, 2, 5, vocab // 2][r % 5]
            off = rng.permutation(vocab)[n:]
            x[r, torch.from_numpy(off)] = math.nan if r % 2 else -math.inf
        for limits in ({}, {"top_k": 3}, {"top_p": 0.9}, {"min_p": 0.1}, {"temperature": 0.0}, {"top_k": 4, "top_p": 0.5}):
            got = check(x, rng.random(20), **limits)
            assert (got[::5] == -1).all() and (got[1::5] >= 0).all()


def set_bits(x, at, bits):
    """Puts the bit pattern `bits` at x[at]."""
    kind, size = {4: (torch.int32, 32), 2: (torch.int16, 16)}[x.element_size()]
    x.view(kind)[at] = bits - (1 << size) if bits >> (size - 1) else bits


# signalling, signalling with its sign set, quiet
NANS = {"f32": (0x7F800001, 0xFFA00000, 0x7FC00000), "f16": (0x7C01, 0xFD00, 0x7E00), "bf16": (0x7F81, 0xFFA0, 0x7FC0)}


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [3007, 66003])
def test_no_nan_hides_what_is_beside_it(vocab, dtype, kind):
    """A NaN at every place of 16 neighbours, the row's largest logit at every other one: in the row's first
    neighbours, in its last ones and between."""
    rng = np.random.default_rng(vocab)
    pairs = [(m, n) for m in range(16) for n in range(16) if m != n]
    x = logits_of(rng, len(pairs), vocab, dtype=dtype)
    most = int(x.float().max()) + 2
    for r, (m, n) in enumerate(pairs):
        first = [0, vocab // 3 // 16 * 16, (vocab - 1) // 16 * 16 - 16][r % 3]
        x[r, first + m] = float(most)
        set_bits(x, (r, first + n), NANS[dtype][kind])
    u = rng.random(len(pairs))
    best = [[0, vocab // 3 // 16 * 16, (vocab - 1) // 16 * 16 - 16][r % 3] + m for r, (m, _) in enumerate(pairs)]
    assert check(x, u, temperature=0.0).tolist() == best and check(x, u, top_k=1).tolist() == best
    for limits in ({"top_k": 3}, {"top_p": 0.5}) + (({}, {"top_p": 0.9}, {"min_p": 0.1}) if vocab < 4000 else ()):
        check(x, u, **limits)


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_rows_of_nans_but_for_a_few(dtype, kind):
    rng = np.random.default_rng(14)
    x = logits_of(rng, 32, 9001, dtype=dtype)
    for r in range(32):
        off = torch.from_numpy(rng.permutation(9001)[[0, 1, 2, 40][r % 4]:])
        set_bits(x, (r, off), NANS[dtype][kind])
    for limits in ({}, {"top_k": 2}, {"top_p": 0.6}, {"min_p": 0.1}, {"temperature": 0.0}):
        got = check(x, rng.random(32), **limits)
        assert (got[::4] == -1).all() and (got[1::4] >= 0).all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_infinite_and_extreme_logits(dtype):
    rng = np.random.default_rng(7)
    x = logits_of(rng, 12, 3001, dtype=dtype)
    most = torch.finfo(TYPES[dtype]).max
    x[0, 17] = math.inf
    x[1, [5, 900, 2999]] = math.inf
    x[2, :] = math.inf
    x[3, 44], x[3, 45] = most, -most
    x[4, :] = -most
    x[5, :] = most
    x[6, ::2] = torch.finfo(TYPES[dtype]).tiny
    x[7, 1::2] = -0.0
    x[7, ::2] = 0.0
    x[8] *= 0
    x[8, 3] = torch.finfo(TYPES[dtype]).smallest_normal / 4
    for limits in ({}, {"top_k": 2}, {"top_k": 2000}, {"top_p": 0.5}, {"top_p": 0.5, "top_k": 2000}, {"min_p": 0.5},
                   {"temperature": 1e-3}, {"temperature": 0.0}):
        check(x, rng.random(12), **limits)
        check(x, np.linspace(0, 1, 12), **limits)


@pytest.mark.parametrize("temperature", [1e-30, 1e-3, 0.05, 30.0, 1e6, 1e30, math.inf])
def test_extreme_temperatures(temperature):
    rng = np.random.default_rng(8)
    for vocab in (100, 20011):
        x = logits_of(rng, 10, vocab)
        for limits in ({}, {"top_k": 30}, {"top_p": 0.6}, {"min_p": 0.3}):
            check(x, rng.random(10), temperature=temperature, **limits)


def test_random_numbers_at_the_ends():
    rng = np.random.default_rng(9)
    x = logits_of(rng, 8, 10007)
    u = np.array([0.0, 2.0**-149, 1e-9, 1 - 2.0**-24, 1.0, 7.0, -1.0, math.nan], np.float32)
    for limits in LIMITS:
        check(x, u, **limits)


def test_values_far_apart():
    """Logits over many orders of magnitude: the bins that look for a border have to shrink to single values."""
    rng = np.random.default_rng(10)
    x = torch.from_numpy((np.sign(rng.normal(size=(10, 6000))) * 10.0 ** rng.uniform(-30, 3, size=(10, 6000))).astype(np.float32))
    for limits in ({"top_k": 100}, {"top_k": 3100}, {"top_p": 0.5}, {"top_p": 0.9, "temperature": 1000.0},
                   {"top_p": 0.7, "temperature": 3e4, "top_k": 5000}):
        check(x, rng.random(10), **limits)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_strides_and_offsets(dtype):
    """Rows that start at any element and lie apart by any distance, also in reverse order of memory."""
    from pynve.torch.nve_sample import sample_tokens

    rng = np.random.default_rng(11)
    base = logits_of(rng, 9, 5003, dtype=dtype).cuda()
    u = torch.rand(9, device="cuda")
    for start, width in ((0, 5003), (1, 5001), (3, 4096), (7, 100), (5, 1)):
        view = base[:, start:start + width]
        for limits in ({}, {"top_k": 20, "top_p": 0.8}, {"top_p": 0.9}):
            a, b = sample_tokens(view, u, **limits), sample_tokens(view.contiguous(), u, **limits)
            assert torch.equal(a, b)
    a, b = sample_tokens(base[::2], u[::2].contiguous(), top_k=5), sample_tokens(base, u, top_k=5)
    assert torch.equal(a, b[::2])
    one = base[:1].expand(9, -1)
    assert torch.equal(sample_tokens(one, u, top_p=0.9), sample_tokens(one.contiguous(), u, top_p=0.9))


def test_no_rows():
    from pynve.torch.nve_sample import sample_tokens

    assert sample_tokens(torch.zeros((0, 50), device="cuda"), torch.zeros(0, device="cuda"), top_k=3).shape == (0,)


def test_rows_past_32_bits():
    """Rows whose elements lie past 2^31 of the first."""
    from pynve.torch.nve_sample import sample_tokens

    rows, vocab = 17000, 131072
    x = torch.zeros((rows, vocab), dtype=torch.float16, device="cuda")
    u = torch.rand(rows, device="cuda")
    last = logits_of(np.random.default_rng(12), 4, vocab, dtype="f16")
    x[-4:] = last.cuda()
    got = sample_tokens(x, u, top_k=9)
    want = R.sample(last.float().numpy(), u[-4:].cpu().numpy(), top_k=9)
    assert got[-4:].tolist() == want.tolist()
    assert torch.equal(got[:-4], (u[:-4].double() * 9).floor().long())


def test_another_stream_and_graph_replays():
    from pynve.torch.nve_sample import sample_tokens

    rng = np.random.default_rng(13)
    x, u = logits_of(rng, 30, 32003).cuda(), torch.rand(30, device="cuda")
    limits = {"temperature": torch.full((30,), 0.8, device="cuda"), "top_k": torch.full((30,), 50, device="cuda").int(),
              "top_p": 0.9}
    want = sample_tokens(x, u, **limits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sample_tokens(x, u, **limits)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sample_tokens(x, u, **limits)
        wide = sample_tokens(x, u, top_p=0.97)
    for i in range(4):
        x.copy_(logits_of(rng, 30, 32003, spread=1.0 + i))
        u.copy_(torch.rand(30))
        limits["top_k"].fill_([50, 0, 3000, 7][i])
        limits["temperature"].fill_([0.8, 1.3, 0.0, 2.0][i])
        graph.replay()
        torch.cuda.synchronize()
        a, b = sample_tokens(x, u, **limits), sample_tokens(x, u, top_p=0.97)
        torch.cuda.synchronize()
        assert torch.equal(got, a) and torch.equal(wide, b)


def test_the_shares_are_the_probabilities():
    """An even grid of random numbers gives every token its probability, to a step of the grid."""
    from pynve.torch.nve_sample import sample_tokens

    n = 4096
    x = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5, 1.5])
    u = (torch.arange(n) + 0.5) / n
    got = torch.bincount(sample_tokens(x.cuda().expand(n, -1), u.cuda(), temperature=0.7).cpu(), minlength=6)
    assert (got - n * torch.softmax(x.double() / 0.7, 0)).abs().max() <= 1.0


def test_traced():
    from pynve.torch.nve_sample import sample_tokens

    x, u = torch.randn(5, 300, device="cuda"), torch.rand(5, device="cuda")
    k = torch.full((5,), 7, device="cuda", dtype=torch.int32)
    f = torch.compile(lambda a, b: sample_tokens(a * 2, b, top_k=k, top_p=0.9), backend="aot_eager", fullgraph=True)
    assert torch.equal(f(x, u), sample_tokens(x * 2, u, top_k=k, top_p=0.9))
    torch.library.opcheck(torch.ops.nve_ops.sample_tokens.default, (x, u, None, k, None, None, 0.5, 0, 0.9, 0.1),
                          test_utils=("test_schema", "test_faketensor"))


def test_refusals():
    from pynve.torch.nve_sample import sample_tokens

    x, u = torch.randn(3, 40, device="cuda"), torch.rand(3, device="cuda")
    f = lambda *s, dtype=torch.float32: torch.ones(s, dtype=dtype, device="cuda")  # noqa: E731

    def run(logits=x, r=u, **limits):
        return sample_tokens(logits, r, **limits)

    run()
    for c in [{"logits": x[0]}, {"logits": x.t()}, {"logits": x[:, :0]}, {"r": u[:2]}, {"r": u.cpu()}, {"r": u[:, None]},
              {"r": f(6)[::2]}, {"temperature": -1.0}, {"temperature": math.nan}, {"top_k": -1}, {"top_k": 1 << 31},
              {"top_p": -0.1}, {"top_p": math.nan}, {"min_p": -0.1}, {"min_p": 1.1}, {"min_p": math.nan},
              {"temperature": f(2)}, {"top_p": f(3).cpu()}, {"min_p": f(3, 1)}]:
        with pytest.raises(ValueError):
            run(**c)
    for c in [{"logits": x.double()}, {"logits": x.long()}, {"r": u.double()}, {"r": u.half()}, {"temperature": f(3).half()},
              {"top_k": f(3)}, {"top_k": f(3, dtype=torch.int64)}]:
        with pytest.raises(TypeError):
            run(**c)
    with pytest.raises(RuntimeError, match="gradient"):
        run(logits=x.clone().requires_grad_())
    with torch.no_grad():
        run(logits=x.clone().requires_grad_())


def check_shares(row, temperature, u):
    """The tokens that `u` draws from `row`, all of whose tokens are kept: a weight may be 2^-31 of itself off, so the
    sums before and up to a token, and u times the total, by as much of the total each; 64-bit sums and series by
    far less than the 2^-41 that are left for them."""
    from pynve.torch.nve_sample import sample_tokens

    got = sample_tokens(row.cuda().expand(len(u), -1), cuda(u), temperature=temperature).cpu().numpy()
    x = row.double().numpy().astype(np.longdouble)
    w = np.exp((x - x.max()) / np.longdouble(np.float32(temperature)))
    after = np.cumsum(w)
    target, room = u.astype(np.longdouble) * after[-1], after[-1] * (2.0**-30 + 2.0**-41)
    assert (w[got] > 0).all()
    low, high = after[got] - w[got] - target, target - after[got]
    assert (low <= room).all() and (high <= room).all(), (float(low.max() / after[-1]), float(high.max() / after[-1]))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("high, small, temperature", [(6.0, 1.93e-5, 1.0), (12.0, 1.93e-5, 0.7), (60.0, 3e-4, 30.0),
                                                      (16.0, 0.011, 1.0), (-3.0, -3.01, 0.01), (700.0, 1.0, 1.0),
                                                      (5000.0, 4990.0, 2.0), (0.0, -1e-3, 1e-4)])
def test_sums_over_16_bit_rows(dtype, high, small, temperature):
    """Logits far smaller than the largest, one of which every 2,048 of the row's first half have."""
    n = 1 << 17
    x = torch.full((n,), small)
    x[:n // 2:2048] = high
    check_shares(x.to(TYPES[dtype]), temperature, ((np.arange(4096) + 0.5) / 4096).astype(np.float32))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("temperature", [1e-6, 0.01, 0.3, 1.0, 7.0, 1000.0])
def test_16_bit_rows_at_any_temperature(dtype, temperature):
    """Magnitudes from 2^-14 to 2^6 of both signs beside a few large logits, units of both kinds."""
    rng = np.random.default_rng(15)
    x = rng.choice([-1.0, 1.0], size=40961) * 2.0 ** rng.uniform(-14, 6, size=40961)
    x[rng.integers(0, 40961, size=30)] = 64.0
    x[20000:24000] = rng.normal(0, 1e-3, size=4000)
    u = np.sort(rng.random(4000)).astype(np.float32)
    check_shares(torch.from_numpy(x).to(TYPES[dtype]), temperature, u)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("temperature", [1e-30, 1e-3, 0.05, 30.0, 1e6, 1e30, math.inf])
def test_extreme_temperatures_of_16_bit_rows(dtype, temperature):
    rng = np.random.default_rng(16)
    x = logits_of(rng, 12, 20011, dtype=dtype)
    x[4:8, ::2] = torch.from_numpy(rng.normal(0, 1e-4, size=(4, 10006)).astype(np.float32)).to(x.dtype)
    x[8:, ::3] = -math.inf
    x[10] -= x[10].max()
    for limits in ({}, {"top_k": 30}, {"top_p": 0.6}, {"min_p": 0.3}):
        check(x, rng.random(12), temperature=temperature, **limits)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("high", [709.0, 711.0, -709.0, -711.0, 0.0])
def test_16_bit_rows_where_the_sums_change(dtype, high):
    """Largest logits on both sides of 1,024 octaves, and weights down to nothing."""
    rng = np.random.default_rng(17)
    x = torch.from_numpy(high - rng.exponential(3.0, size=30011)).to(TYPES[dtype])
    x[::7] = high - 900.0
    x[5] = high
    check_shares(x, 1.0, np.sort(rng.random(2000)).astype(np.float32))
