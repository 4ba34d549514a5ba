"""The operators of the key-value cache together, as examples/sequence_decode.py
uses them behind an embedding layer: the decoded rows against the same model
computed whole in 64 bits, and a run whose caches are cut to their budget."""
import os
import sys

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def whole(m, history):
    """The hidden rows of the last item of every user, from the whole history [steps, users], in 64 bits."""
    n = torch.nn.functional
    steps = history.shape[0]
    x = m.emb.weight.data[history].double().cpu()  # [steps, users, width]
    cos, sin = (t.double().cpu()[:steps, None, None] for t in m.cos_sin.split(m.dim // 2, 1))
    turn = lambda t: torch.cat([t[..., :m.dim // 2] * cos - t[..., m.dim // 2:] * sin,  # noqa: E731
                                t[..., m.dim // 2:] * cos + t[..., :m.dim // 2] * sin], -1)
    mask = torch.full((steps, steps), float("-inf"), dtype=torch.float64).triu(1)
    for w in m.blocks:
        w = {k: t.double().cpu() for k, t in w.items()}
        qkv = (n.layer_norm(x, x.shape[2:]) @ w["qkv"]).view(steps, x.shape[1], -1, m.dim)
        q, k, v = qkv.split([m.q_heads, m.kv_heads, m.kv_heads], 2)
        group = m.q_heads // m.kv_heads
        q, k, v = turn(q), turn(k).repeat_interleave(group, 2), v.repeat_interleave(group, 2)
        q, k, v = (t.permute(1, 2, 0, 3) for t in (q, k, v))  # [users, heads, steps, dim]
        p = torch.softmax(q @ k.transpose(2, 3) * m.dim**-0.5 + mask, -1)
        x = x + (p @ v).permute(2, 0, 1, 3).flatten(2) @ w["out"]
        x = x + n.gelu(n.layer_norm(x, x.shape[2:]) @ w["up"]) @ w["down"]
    return x[-1]


def test_decoded_rows_match_the_whole_model():
    """In f32 a product of up to 512 terms, two blocks deep, is some 1e-6 off; 1e-4 leaves room for the norms."""
    from sequence_decode import SequenceDecoder

    m = SequenceDecoder(1000, 5, budget=64, longest=50, dtype=torch.float32)
    history = torch.randint(0, 1000, (40, 5), device="cuda")
    for row in history:
        got = m.step(row)
    want = whole(m, history.cpu().to("cuda"))
    assert (got.double().cpu() - want).abs().max() <= 1e-4 * want.abs().max()


@pytest.mark.parametrize("args", [["--users", "3", "--steps", "90", "--budget", "32", "--items", "500"],
                                  ["--users", "7", "--steps", "60", "--budget", "16", "--items", "2000", "--e4m3"]])
def test_the_example_runs_within_its_budget(args, capsys):
    import sequence_decode

    items = sequence_decode.main(args)
    assert items.shape == (int(args[1]),)
    kept = int(capsys.readouterr().out.split(" of ")[0].split()[-1])
    assert int(args[5]) <= kept < int(args[5]) + 16


def test_evicted_caches_keep_the_first_and_the_latest():
    from sequence_decode import SequenceDecoder

    m = SequenceDecoder(1000, 4, budget=48, sinks=3, recent=20, longest=200)
    for _ in range(48 + 16 * 3 + 5):
        out = m.step(torch.randint(0, 1000, (4,), device="cuda"))
    assert torch.isfinite(out).all() and m.length == 48 + 5
    for cache in m.caches:
        for user in range(4):
            pages = m.tables[user].long()
            held = cache.index[pages].transpose(0, 1).flatten(1)[:, :m.length]
            for head in held.cpu().tolist():
                assert len(set(head)) == m.length
                # what was protected when the cache was last cut, and what came after
                assert set(range(3)) <= set(head) and set(range(m.seen - 5 - 20, m.seen)) <= set(head)
