"""The operators of the paged key-value cache that are timed: which calls, at which sizes, on which values.

A model that answers one token at a time keeps the keys and values of its
attention in pages of `page` slots.  Three operators work on them:

  append   pynve.torch.nve_kv.kv_append: rotates the new tokens' queries and keys by their positions
           (one axis for text; time, height and width for images and video), writes keys and values
  attend   pynve.torch.nve_kv.kv_attend: attention of one new token per sequence over its pages; with
           `track`, each slot's attention weight is added to the weight the cache holds for it
  evict    pynve.torch.nve_kv.kv_evict: every sequence longer than `budget` drops the slots of the least
           accumulated weight, and the kept ones close the gaps

Where `own` is false, `run` computes the same with elementary torch operations in 32 bits.
"""
import math
import os
import random
import sys

import torch

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(_ROOT, "nv-embedding-cache_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

_TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
_E4M3_MAX = 448.0
_TINY = 1e-30  # the least largest magnitude an e4m3 row's scale is made for


def _case(op, **fields):
    """Every case has the same fields, so that a new one is a change of values only."""
    c = {"op": op, "dtype": "bf16", "cache": "", "seqs": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "shortest": 0, "longest": 0, "track": False, "fused": False, "tokens": 0, "axes": 1, "rot": 0,
         "interleaved": False, "budget": 0, "sinks": 0, "recent": 0, "used": False}
    c.update(fields)
    c["cache"] = c["cache"] or c["dtype"]
    c["shortest"] = c["shortest"] or c["longest"]
    return c


def listed():
    named = {
        # one user's conversation: a single sequence, latency counts
        "attend_request": _case("attend", longest=777),
        # a serving batch of sequences of very different lengths under a budgeted cache
        "attend_batch": _case("attend", seqs=64, shortest=512, longest=8192, track=True, fused=True),
        # one very long document: all parallelism has to come from its length
        "attend_long": _case("attend", dtype="f16", longest=200001),
        # a large batch over an 8-bit cache, wide groups
        "attend_e4m3": _case("attend", cache="e4m3", seqs=256, q_heads=64, shortest=200, longest=4096, page=64),
        # user histories of a sequence recommender in 32 bits, a key head for each query head
        "attend_f32": _case("attend", dtype="f32", seqs=48, q_heads=12, kv_heads=12, dim=64, shortest=1, longest=2000,
                            page=32, track=True),
        # a head width and a group that are no powers of two, few key heads, small pages
        "attend_odd": _case("attend", dtype="f16", seqs=7, q_heads=20, kv_heads=2, dim=80, shortest=33, longest=30011,
                            page=8, track=True, fused=True),
        # one decode step of a batch
        "append_step": _case("append", seqs=64, longest=1024, tokens=64, rot=128, fused=True),
        # a video's tokens enter the cache: positions in time, height and width
        "append_video": _case("append", dtype="f16", longest=16001, tokens=16001, axes=3, rot=128, fused=True),
        # a prompt enters an 8-bit cache; part of each head is rotated, neighbours as pairs
        "append_e4m3": _case("append", cache="e4m3", seqs=3, longest=3000, tokens=9000, dim=96, rot=64,
                             interleaved=True, page=64),
        # a serving batch in the steady state: one page too many
        "evict_step": _case("evict", seqs=64, longest=2064, budget=2048, sinks=4, recent=256, used=True),
        # after long prompts: an eighth is kept
        "evict_prompt": _case("evict", dtype="f16", seqs=8, longest=32768, budget=4096, sinks=4, recent=512),
        # sequences of different lengths, some within the budget, in an 8-bit cache
        "evict_e4m3": _case("evict", cache="e4m3", seqs=33, kv_heads=5, dim=96, shortest=20, longest=12000,
                            page=64, budget=1000, recent=100, used=True),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["attend", "attend", "append", "evict"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    cache = "e4m3" if dtype != "f32" and rng.random() < 0.3 else dtype
    kv = rng.choice([1, 2, 3, 4, 5, 8, 8, 12, 16])
    dim = rng.choice([64, 128, 128, 8 * rng.randint(2, 32)])
    c = _case(op, dtype=dtype, cache=cache, kv_heads=kv, q_heads=kv * rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 8, 12, 16, 24]),
              dim=dim, page=rng.choice([8, 16, 16, 32, 64, 128, 256]), seqs=_log(rng, 1, 256),
              longest=_log(rng, 1, 131072), fused=rng.random() < 0.5)
    c["shortest"] = c["longest"] if rng.random() < 0.3 else _log(rng, 1, c["longest"])
    if op == "attend":
        c["track"] = rng.random() < 0.5
    elif op == "append":
        c["tokens"] = _log(rng, 1, min(32768, sum(_lengths(c))))
        c["axes"] = rng.choice([1, 1, 2, 3])
        c["rot"] = rng.choice([dim, dim, dim // 2 // 2 * 2, 0])
        c["interleaved"] = rng.random() < 0.5
    else:
        c["budget"] = _log(rng, 1, c["longest"])
        c["sinks"] = rng.choice([0, 4, 16])
        c["recent"] = rng.choice([0, c["budget"] // 8, c["budget"] // 2])
        c["used"] = rng.random() < 0.5
    return c


def draw(rng):
    """A case of the same kinds: any type, head layout and page, from one slot to the longest cache."""
    most = max(work(c)["bytes"] for c in listed())
    while True:
        c = _draw(rng)
        rows = c["seqs"] * c["kv_heads"] * c["longest"]
        if c["op"] == "append" and c["rot"] == 0:
            c["axes"], c["interleaved"] = 1, False
        # the plain form pads to the longest sequence and widens to 32 bits
        wide = rows * c["dim"] * 4 <= 3 << 30 and c["seqs"] * c["q_heads"] * c["longest"] * 4 <= 1 << 30
        if work(c)["bytes"] <= most and wide and sum(_lengths(c)) * c["kv_heads"] * c["dim"] * 2 <= 3 << 30:
            return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(c):
    """The sequences' lengths, ascending: evenly spread in their logarithm, so the same for every seed."""
    n, lo, hi = c["seqs"], math.log(c["shortest"]), math.log(c["longest"])
    return [int(round(math.exp(hi if n == 1 else lo + (hi - lo) * i / (n - 1)))) for i in range(n)]


def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 16 + what)
    return g


def _normal(shape, dtype, gen, scale=1.0):
    t = torch.empty(shape, device="cuda", dtype=dtype)
    return t.normal_(0.0, scale, generator=gen)


def _heads(c, rows, gen, scale):
    """q, k and v of `rows` tokens [rows, heads, dim]: slices of one projection's output where `fused`."""
    dt, hq, hk, d = _TORCH[c["dtype"]], c["q_heads"], c["kv_heads"], c["dim"]
    x = _normal((rows, hq + 2 * hk, d), dt, gen)
    x[:, :hq] *= scale
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    return (q, k, v) if c["fused"] else (q.contiguous(), k.contiguous(), v.contiguous())


def _pages(c, gen, num_pages):
    """Random rows of the cache's type [num_pages, kv_heads, page, dim] and, for e4m3, their scales."""
    shape = (num_pages, c["kv_heads"], c["page"], c["dim"])
    if c["cache"] != "e4m3":
        return _normal(shape, _TORCH[c["cache"]], gen), None
    x = _normal(shape, torch.float16, gen)
    scale = x.abs().amax(-1).float() / _E4M3_MAX
    return (x / scale.unsqueeze(-1)).clamp_(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn), scale


def _rotary(c):
    """cos and sin [positions, rot] for the positions that occur: the usual geometric frequencies."""
    n = c["longest"] + 1
    f = torch.pow(10000.0, -torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float()


def _sections(c):
    """Pairs per axis: the first axis has what the others leave."""
    each = c["rot"] // 2 // c["axes"]
    return [c["rot"] // 2 - each * (c["axes"] - 1)] + [each] * (c["axes"] - 1)


def prepare(case, seed):
    c, page = case, case["page"]
    g = _gen(seed, 1)
    lengths = torch.tensor(_lengths(c), device="cuda", dtype=torch.int32)
    lengths = lengths[torch.randperm(c["seqs"], device="cuda", generator=g)]
    counts = (lengths + page - 1) // page
    per_seq = -(-c["longest"] // page)
    num_pages = sum(-(-n // page) for n in _lengths(c)) + 1
    # every sequence has pages of its own, anywhere in the cache; entries past its last page hold a spare page
    spread = torch.randperm(num_pages, device="cuda", generator=g).int()
    table = torch.full((c["seqs"], per_seq), int(spread[-1]), device="cuda", dtype=torch.int32)
    used = torch.arange(per_seq, device="cuda") < counts[:, None]
    table[used] = spread[:-1]
    k, k_scale = _pages(c, _gen(seed, 2), num_pages)
    v, v_scale = _pages(c, _gen(seed, 3), num_pages)
    s = {"case": c, "lengths": lengths, "table": table, "k_pages": k, "v_pages": v, "k_scale": k_scale,
         "v_scale": v_scale, "weights": None}
    shape = (num_pages, c["kv_heads"], page)
    if c["op"] == "attend":
        # queries wide enough that a few slots carry most of the weight, as trained models have
        s["q"] = _heads(c, c["seqs"], _gen(seed, 4), 3.0)[0]
        s["scale"] = c["dim"] ** -0.5
        if c["track"]:
            s["weights"] = torch.rand(shape, device="cuda", generator=g)
        return s
    if c["op"] == "append":
        n = c["tokens"]
        s["q"], s["k"], s["v"] = _heads(c, n, _gen(seed, 4), 1.0)
        # the last tokens of the sequences, in the sequences' order
        at = torch.arange(n, device="cuda")
        ends = torch.cumsum(lengths.long(), 0)
        flat = (ends[-1] - n + at).clamp_(min=0)
        seq = torch.searchsorted(ends, flat, right=True)
        place = flat - (ends - lengths)[seq]
        if n <= c["seqs"]:  # a decode step: one token per sequence
            seq = torch.randperm(c["seqs"], device="cuda", generator=g)[:n]
            place = lengths.long()[seq] - 1
        s["slots"] = table[seq, place // page].long() * page + place % page
        s["index"] = place.int()
        s["index_pages"] = torch.zeros(shape, device="cuda", dtype=torch.int32)
        s["weights"] = torch.rand(shape, device="cuda", generator=g)
        if c["rot"]:
            s["cos_sin"], s["sections"] = _rotary(c), _sections(c)
            rows = [place.int()] + [torch.randint(0, min(64, c["longest"]), (n,), device="cuda", generator=g).int()
                                    for _ in range(c["axes"] - 1)]
            s["positions"] = torch.stack(rows)
        return s
    # weights of a heavy-tailed distribution, some of them zero; after earlier evictions the slots are in any order
    w = torch.exp(2.0 * _normal(shape, torch.float32, g))
    s["fresh"] = w * (torch.rand(shape, device="cuda", generator=g) > 0.02)
    s["weights"] = torch.empty_like(w)
    place = torch.arange(per_seq * page, device="cuda", dtype=torch.int32)
    if c["used"]:
        place = place.view(per_seq, page).t().reshape(-1)  # spread over the pages
    index = torch.zeros(shape, device="cuda", dtype=torch.int32)
    rows = place.view(per_seq, 1, page).expand(per_seq, c["kv_heads"], page)
    index[table[used].long()] = rows.expand(c["seqs"], *rows.shape)[used]
    s["index_pages"] = index
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _gather(s, pages, scale):
    """The pages of every sequence as [seqs, kv_heads, slots, ...] in 32 bits, padded to the longest."""
    x = pages[s["table"].long()].float()
    if scale is not None:
        x = x * scale[s["table"].long()].unsqueeze(-1)
    return x.transpose(1, 2).flatten(2, 3)


def _inside(s):
    """[seqs, slots]: the slots below each sequence's length."""
    n = s["table"].shape[1] * s["case"]["page"]
    return torch.arange(n, device="cuda") < s["lengths"][:, None]


def _attend(s):
    c, inside = s["case"], _inside(s)
    n, hk, d = c["seqs"], c["kv_heads"], c["dim"]
    q = s["q"].float().reshape(n, hk, c["q_heads"] // hk, d)
    k = _gather(s, s["k_pages"], s["k_scale"])
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    x = x.masked_fill(~inside[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    v = _gather(s, s["v_pages"], s["v_scale"]).masked_fill(~inside[:, None, :, None], 0.0)
    out = torch.matmul(x, v).reshape(n, c["q_heads"], d).to(s["q"].dtype)
    if not c["track"]:
        return {"out": out}
    w = s["weights"].transpose(0, 1).clone().flatten(1)  # [kv_heads, slots]
    rows = (s["table"].long()[:, :, None] * c["page"] + torch.arange(c["page"], device="cuda")).flatten(1)[inside]
    w[:, rows] = w[:, rows] + x.sum(2).transpose(0, 1)[:, inside]
    s["weights"].copy_(w.view(hk, -1, c["page"]).transpose(0, 1))
    return {"out": out, "weights": s["weights"]}


def _rotate(s, x):
    """The rotated rows of x [tokens, heads, dim] in 32 bits."""
    c, x = s["case"], x.float()
    if not c["rot"]:
        return x
    r, half = c["rot"], c["rot"] // 2
    # the position of every pair's axis: [tokens, pairs]
    at = torch.cat([p[:, None].expand(-1, n) for p, n in zip(s["positions"].long(), s["sections"])], 1)
    pair = torch.arange(half, device="cuda")
    cos, sin = s["cos_sin"][at, pair].unsqueeze(1), s["cos_sin"][at, pair + half].unsqueeze(1)
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if c["interleaved"] else (x[..., :half], x[..., half:r])
    y = [a * cos - b * sin, b * cos + a * sin]
    y = torch.stack(y, -1).flatten(-2) if c["interleaved"] else torch.cat(y, -1)
    return torch.cat([y, x[..., r:]], -1)


def _store(s, pages, scales, x):
    page = s["case"]["page"]
    at = (s["slots"] // page, slice(None), s["slots"] % page)
    if scales is None:
        pages[at] = x.to(pages.dtype)
        return
    scale = x.abs().amax(-1).clamp(min=_TINY) / _E4M3_MAX
    scales[at] = scale
    codes = (x / scale.unsqueeze(-1)).to(torch.float8_e4m3fn)
    pages.view(torch.uint8)[at] = codes.view(torch.uint8)


def _append(s):
    q = _rotate(s, s["q"]).to(s["q"].dtype)
    _store(s, s["k_pages"], s["k_scale"], _rotate(s, s["k"]))
    _store(s, s["v_pages"], s["v_scale"], s["v"].float())
    page = s["case"]["page"]
    at = (s["slots"] // page, slice(None), s["slots"] % page)
    s["index_pages"][at] = s["index"][:, None].expand(-1, s["case"]["kv_heads"])
    s["weights"][at] = 0.0
    return q


def _evict(s):
    c, inside = s["case"], _inside(s)
    hk, page, n = c["kv_heads"], c["page"], s["table"].shape[1] * c["page"]
    keep = torch.minimum(s["lengths"], torch.tensor(c["budget"], device="cuda", dtype=torch.int32))
    at = s["table"].long()
    w = s["weights"][at].transpose(1, 2).flatten(2)  # [seqs, kv_heads, slots]
    index = s["index_pages"][at].transpose(1, 2).flatten(2)
    newest = index.masked_fill(~inside[:, None], -1).amax(-1, keepdim=True)
    held = (index < c["sinks"]) | (index > newest - c["recent"])
    # ascending in (outside, protected, weight, slot): the first length - budget of those inside are dropped
    order = torch.argsort(w, dim=-1, stable=True)
    rank = held.int() + 2 * (~inside[:, None]).int()
    order = order.gather(-1, torch.argsort(rank.gather(-1, order), dim=-1, stable=True))
    place = torch.empty_like(order).scatter_(-1, order, torch.arange(n, device="cuda").expand_as(order).contiguous())
    dropped = place < (s["lengths"] - keep)[:, None, None]
    below = torch.arange(n, device="cuda") < keep[:, None, None]
    hole = dropped & below
    moved = ~dropped & ~below & inside[:, None]
    # the j-th hole of a head takes the row of its j-th kept slot past the budget
    row = (at[:, None, :, None] * hk + torch.arange(hk, device="cuda")[:, None, None]) * page
    row = (row + torch.arange(page, device="cuda")).flatten(2)
    to, of = row[hole], row[moved]
    for name in ("k_pages", "v_pages"):
        x = s[name].view(torch.uint8) if c["cache"] == "e4m3" else s[name]
        x = x.view(-1, c["dim"])
        x[to] = x[of]
    for name in ("k_scale", "v_scale", "weights", "index_pages"):
        if s[name] is not None:
            x = s[name].view(-1)
            x[to] = x[of]
    return keep


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _written(s, first):
    """What an operator gives back or changes: its own answer and the cache."""
    keys = ("k_pages", "v_pages", "k_scale", "v_scale", "weights", "index_pages")
    return {"answer": first, **{k: s[k] for k in keys if s[k] is not None}}


def run(state):
    s, c = state, state["case"]
    if c["op"] == "evict":  # since the last eviction the attention has added to the weights
        s["weights"].copy_(s["fresh"])
    if not own:
        if c["op"] == "attend":
            return _attend(s)
        return _written(s, _append(s) if c["op"] == "append" else _evict(s))
    from pynve.torch import nve_kv

    if c["op"] == "attend":
        out = nve_kv.kv_attend(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], scale=s["scale"],
                               k_scale=s["k_scale"], v_scale=s["v_scale"], weights=s["weights"])
        return {"out": out, "weights": s["weights"]} if c["track"] else {"out": out}
    if c["op"] == "append":
        q = nve_kv.kv_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"], q=s["q"],
                             positions=s.get("positions"), cos_sin=s.get("cos_sin"), sections=s.get("sections"),
                             interleaved=c["interleaved"], index=s["index"], k_scale=s["k_scale"],
                             v_scale=s["v_scale"], weights=s["weights"], index_pages=s["index_pages"])
        return _written(s, q)
    n = nve_kv.kv_evict(s["k_pages"], s["v_pages"], s["weights"], s["index_pages"], s["table"], s["lengths"],
                        c["budget"], sinks=c["sinks"], recent=c["recent"], k_scale=s["k_scale"],
                        v_scale=s["v_scale"])
    return _written(s, n)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c, lengths = case, _lengths(case)
    row = c["dim"] * _SIZE[c["cache"]] + (4 if c["cache"] == "e4m3" else 0)
    hq, hk, d, e = c["q_heads"], c["kv_heads"], c["dim"], _SIZE[c["dtype"]]
    if c["op"] == "attend":
        slots = sum(lengths)
        total = slots * hk * 2 * row + 2 * c["seqs"] * hq * d * e + 4 * sum(-(-n // c["page"]) for n in lengths)
        total += 8 * slots * hk if c["track"] else 0
        return {"bytes": float(total), "flops": 4.0 * slots * hq * d}
    if c["op"] == "append":
        n = c["tokens"]
        total = n * ((2 * hq + 2 * hk) * d * e + 2 * hk * row + 8 * hk + 12 + 4 * c["rot"] + 4 * c["axes"])
        return {"bytes": float(total), "flops": 3.0 * n * (hq + hk) * c["rot"]}
    # the weights as they have become (read and written), weights and places read, the kept rows past the budget moved
    total = 8 * sum(lengths) * hk
    for n in lengths:
        if n > c["budget"]:
            total += 8 * n * hk + 2 * hk * (2 * row + 8) * c["budget"] * (n - c["budget"]) / n
    return {"bytes": float(total), "flops": 0.0}


# ---------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------
def _rows64(s, name, seq, head):
    """One head's rows of a sequence in 64 bits."""
    n = int(s["lengths"][seq])
    slot = torch.arange(n, device="cuda")
    p, o = s["table"][seq].long()[slot // s["case"]["page"]], slot % s["case"]["page"]
    x = s[name + "_pages"][p, head, o].double()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][p, head, o].double().unsqueeze(-1)
    return x, p, o


def _attend64(s):
    c = s["case"]
    group = c["q_heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    weights = None if s["weights"] is None else s["weights"].double()
    for i in range(c["seqs"]):
        for h in range(c["kv_heads"]):
            heads = slice(h * group, (h + 1) * group)
            k, p, o = _rows64(s, "k", i, h)
            v = _rows64(s, "v", i, h)[0]
            a = torch.softmax(torch.mm(s["q"][i, heads].double(), k.t().contiguous()) * s["scale"], -1)
            out[i, heads] = torch.mm(a, v)
            if weights is not None:
                weights[p, h, o] += a.sum(0)
    return {"out": out} if weights is None else {"out": out, "weights": weights}


def _rotate64(s, x):
    c = s["case"]
    y = x.double().clone()
    pair = 0
    for axis, pairs in enumerate(s["sections"] if c["rot"] else []):
        row = s["cos_sin"][s["positions"][axis].long()].double()
        for i in range(pair, pair + pairs):
            a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + c["rot"] // 2)
            co, si = row[:, None, i], row[:, None, i + c["rot"] // 2]
            y[..., a] = x[..., a].double() * co - x[..., b].double() * si
            y[..., b] = x[..., a].double() * si + x[..., b].double() * co
        pair += pairs
    return y


def _append64(s):
    page = s["case"]["page"]
    p, o = s["slots"] // page, s["slots"] % page
    got = {"answer": _rotate64(s, s["q"]), "weights": s["weights"].double(), "index_pages": s["index_pages"]}
    got["weights"][p, :, o] = 0.0
    got["index_pages"][p, :, o] = s["index"][:, None]
    for name, x in (("k", _rotate64(s, s["k"])), ("v", s["v"].double())):
        pages = s[name + "_pages"].double()
        if s[name + "_scale"] is not None:
            scale = x.abs().amax(-1).clamp(min=_TINY) / _E4M3_MAX
            got[name + "_scale"] = s[name + "_scale"].double()
            got[name + "_scale"][p, :, o] = scale
            x = x / scale.unsqueeze(-1)
        pages[p, :, o] = x
        got[name + "_pages"] = pages
    return got


def exact(case, seed):
    c = case
    if c["op"] == "evict":  # rows are moved as they are: nothing is computed
        return None
    if c["op"] == "attend" and c["seqs"] * c["kv_heads"] > 4096:
        return None
    s = prepare(c, seed)
    return _attend64(s) if c["op"] == "attend" else _append64(s)


if __name__ == "__main__":
    for _c in listed() + [draw(random.Random(1))]:
        print(_c.get("name", "drawn"), work(_c))
