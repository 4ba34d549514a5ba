"""The decoder's operators together, as examples/sequence_decode.py uses them: 4-bit caches, normed heads and
drawn items, step by step against the same steps restated, and the example's own runs."""
import os
import sys

import numpy as np
import pytest

import kv4_reference as R4
import sample_reference as RS

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def whole(m, history):
    """The hidden rows of the last item of every user, from the whole history [steps, users], in 64 bits; normed heads."""
    n = torch.nn.functional
    steps = history.shape[0]
    x = m.emb.weight.data[history].double().cpu()
    cos, sin = (t.double().cpu()[:steps, None, None] for t in m.cos_sin.split(m.dim // 2, 1))
    half = m.dim // 2
    turn = lambda t: torch.cat([t[..., :half] * cos - t[..., half:] * sin,  # noqa: E731
                                t[..., half:] * cos + t[..., :half] * sin], -1)
    norm = lambda t, w: t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731
    mask = torch.full((steps, steps), float("-inf"), dtype=torch.float64).triu(1)
    for w in m.blocks:
        w = {k: t.double().cpu() for k, t in w.items()}
        qkv = (n.layer_norm(x, x.shape[2:]) @ w["qkv"]).view(steps, x.shape[1], -1, m.dim)
        q, k, v = qkv.split([m.q_heads, m.kv_heads, m.kv_heads], 2)
        group = m.q_heads // m.kv_heads
        q, k = turn(norm(q, w["q_norm"])), turn(norm(k, w["k_norm"])).repeat_interleave(group, 2)
        q, k, v = (t.permute(1, 2, 0, 3) for t in (q, k, v.repeat_interleave(group, 2)))
        p = torch.softmax(q @ k.transpose(2, 3) * m.dim**-0.5 + mask, -1)
        x = x + (p @ v).permute(2, 0, 1, 3).flatten(2) @ w["out"]
        x = x + n.gelu(n.layer_norm(x, x.shape[2:]) @ w["up"]) @ w["down"]
    return x[-1]


def test_normed_rows_match_the_whole_model():
    """In f32 a product of up to 512 terms, two blocks deep, is some 1e-6 off; 1e-4 leaves room for the norms."""
    from sequence_decode import SequenceDecoder

    m = SequenceDecoder(1000, 5, budget=64, longest=50, dtype=torch.float32, norms=True)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    for w in m.blocks:
        for name in ("q_norm", "k_norm"):
            w[name].copy_(0.5 + torch.rand(m.dim, device="cuda", generator=g))
    history = torch.randint(0, 1000, (40, 5), device="cuda")
    for row in history:
        got = m.step(row)
    want = whole(m, history.cpu().to("cuda"))
    assert (got.double().cpu() - want).abs().max() <= 1e-4 * want.abs().max()


def test_drawn_items_are_the_restated_draws():
    """A cache of 4 bits, items drawn from the scores that the step gives: each draw is the definition's."""
    from sequence_decode import SequenceDecoder

    users = 6
    m = SequenceDecoder(700, users, budget=32, longest=90, cache_dtype=torch.float4_e2m1fn_x2, norms=True)
    candidates = torch.arange(0, 700, 3, device="cuda")
    items = torch.randint(0, 700, (users,), device="cuda")
    for step in range(70):  # past the budget: rows are evicted
        hidden = m.step(items)
        u = torch.rand(users, device="cuda")
        limits = [{"temperature": 0.7, "top_k": 20}, {"top_p": 0.8}, {"min_p": 0.1, "temperature": 1.5}][step % 3]
        items = m.next_items(hidden, candidates, u, **limits)
        scores = (hidden @ m.emb(candidates).t()).float().cpu().numpy()
        want = RS.sample(scores, u.cpu().numpy(), **limits)
        assert items.tolist() == candidates.cpu()[torch.from_numpy(want)].tolist()
    assert torch.isfinite(hidden).all() and 32 <= m.length < 48
    # what the caches hold are codes and scales as they come from rows: no scale is a NaN's
    for cache in m.caches:
        assert np.isfinite(R4.values64(cache.k.view(torch.uint8).cpu(), cache.k_scale.view(torch.uint8).cpu())).all()


@pytest.mark.parametrize("args", [["--users", "3", "--steps", "90", "--budget", "32", "--items", "500", "--mxfp4"],
                                  ["--users", "7", "--steps", "60", "--budget", "16", "--items", "2000", "--mxfp4", "--norms",
                                   "--temperature", "0.8", "--top-k", "50", "--top-p", "0.9", "--min-p", "0.01"],
                                  ["--users", "2", "--steps", "20", "--budget", "16", "--items", "300", "--norms",
                                   "--temperature", "1.0"]])
def test_the_example_runs_within_its_budget(args, capsys):
    import sequence_decode

    items = sequence_decode.main(args)
    assert items.shape == (int(args[1]),) and ((items >= 0) & (items < int(args[7]))).all()
    kept = int(capsys.readouterr().out.split(" of ")[0].split()[-1])
    assert kept < int(args[5]) + 16
