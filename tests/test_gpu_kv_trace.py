"""The paged key-value cache's operators under tracing: a step of append, attend and evict gives the
compiled program's results and cache as it does by itself, and the schemas say what is written."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def state(cache=torch.float16):
    from pynve.torch.nve_kv import KVCache

    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    c = KVCache(12, 2, 64, dtype=cache)
    table = torch.randperm(12, device="cuda", generator=g).int().view(3, 4)
    n = 150
    rows = lambda heads, n: torch.randn(n, heads, 64, device="cuda", generator=g).half()  # noqa: E731
    seq = torch.arange(n, device="cuda") % 3
    place = torch.arange(n, device="cuda") // 3
    c.append(rows(2, n), rows(2, n), c.slots(table, seq, place), index=place.int())
    lengths = torch.full((3,), 51, device="cuda", dtype=torch.int32)
    slots = c.slots(table, torch.arange(3, device="cuda"), torch.full((3,), 50, device="cuda"))
    angle = torch.rand(60, 32, device="cuda", generator=g)
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1)
    return c, (rows(8, 3), rows(2, 3), rows(2, 3), slots, table, lengths, lengths - 1, cos_sin)


def step(c, q, k, v, slots, table, lengths, at, cos_sin):
    q = c.append(k, v, slots, q=q, positions=at, cos_sin=cos_sin)
    out, lse = c.attend(q, table, lengths, return_lse=True)
    return q, out, lse, c.evict(table, lengths, 40, sinks=2, recent=8)


@pytest.mark.parametrize("cache", [torch.float16, torch.float8_e4m3fn])
def test_a_compiled_step(cache):
    a, b = state(cache), state(cache)
    want = step(a[0], *a[1])
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(b[0], *b[1])
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    bits = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t  # noqa: E731
    for name in ("k", "v", "k_scale", "v_scale", "weights", "index"):
        x, y = getattr(b[0], name), getattr(a[0], name)
        assert x is y is None or torch.equal(bits(x), bits(y)), name


def test_schemas_say_what_is_written():
    c, (q, k, v, slots, table, lengths, at, cos_sin) = state()
    check = {"test_utils": ("test_schema", "test_faketensor")}
    ops = torch.ops.nve_ops
    torch.library.opcheck(ops.kv_append.default, (k, v, c.k, c.v, slots, q, at, cos_sin, None, False, None, None, None,
                                                  c.weights, c.index), **check)
    torch.library.opcheck(ops.kv_append.default, (k, v, c.k, c.v, slots, None, None, None, None, False, None, None, None,
                                                  None, None), **check)
    for op in (ops.kv_attend.default, ops.kv_attend_lse.default):
        torch.library.opcheck(op, (q, c.k, c.v, table, lengths, 0.125, None, None, c.weights, 0), **check)
        torch.library.opcheck(op, (q, c.k, c.v, table, lengths, 0.125, None, None, None, 60), **check)
    torch.library.opcheck(ops.kv_evict.default, (c.k, c.v, c.weights, c.index, table, lengths, 40, 2, 8, None, None),
                          **check)
