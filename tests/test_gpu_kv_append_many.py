"""Appends of more tokens than one launch has threads for (2^32 of them): nearly all slots lie outside
the cache, the others are around the places where launches may meet."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def run(tokens, dim, rot, offset):
    from pynve.torch import nve_kv

    page = 16
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens)
    at = sorted({0, 1, tokens // 2 - 1, tokens // 2, tokens - 1} |
                {t for edge in range(1 << 22, tokens, 1 << 22) for t in (edge - 9, edge - 8, edge - 1, edge)})
    picked = torch.tensor(at, device="cuda")
    num_pages = -(-len(at) // page)
    slots = torch.full((tokens,), -1, dtype=torch.int64, device="cuda")
    slots[picked] = torch.arange(len(at), device="cuda")
    # every token's rows are the same, which takes no memory: the index tells the tokens apart
    base = torch.randn(2, dim + 8, device="cuda", generator=g).half()
    k, v = (row[offset:offset + dim].expand(tokens, 1, dim) for row in base)
    positions = cos_sin = None
    if rot:
        positions = torch.arange(tokens, device="cuda", dtype=torch.int32).remainder_(7)
        cos_sin = torch.randn(7, rot, device="cuda", generator=g)
    index = torch.arange(tokens, device="cuda", dtype=torch.int32)

    def append(rows, k, v, positions, index):
        pages = [torch.zeros((num_pages, 1, page, dim), dtype=torch.float16, device="cuda") for _ in range(2)]
        weights = torch.ones((num_pages, 1, page), device="cuda")
        places = torch.zeros((num_pages, 1, page), dtype=torch.int32, device="cuda")
        nve_kv.kv_append(k, v, *pages, rows, positions=positions, cos_sin=cos_sin, index=index, weights=weights,
                         index_pages=places)
        return pages + [weights, places]

    got = append(slots, k, v, positions, index)
    want = append(slots[picked], k[:len(at)], v[:len(at)], None if positions is None else positions[picked],
                  index[picked])
    torch.cuda.synchronize()
    assert want[3].flatten()[:len(at)].tolist() == at
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_a_value_a_lane():
    """A wave a head row: 2^26 + 10 rows, which start off 16 bytes."""
    run((1 << 25) + 5, 8, 0, 1)


def test_16_values_a_lane():
    """8 tokens a workgroup of 256 threads: 2^27 + 100 tokens."""
    run((1 << 27) + 100, 256, 256, 0)
