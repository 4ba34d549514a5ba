"""Plain restatements of the paged key-value cache's operators, on the CPU, for
the tests: attention in 64 bits with the error bounds its kernel has to keep,
append in the f32 steps its definition names, eviction by sorting."""
import math

import numpy as np
import torch

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
# half a unit in the last place, relative
HALF_ULP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
# least magnitude a type's rounding is relative for (half its spacing below that is absolute)
SMALL = {"f32": 2.0**-126, "f16": 2.0**-14, "bf16": 2.0**-126}


def make_pages(dtype, num_pages, heads, page, dim, rng, spread=1.0):
    """Random pages (CPU) and, for e4m3, their scales."""
    x = torch.from_numpy(rng.normal(0, spread, size=(num_pages, heads, page, dim)).astype(np.float32))
    if dtype != "e4m3":
        return x.to(TORCH[dtype]), None
    scale = x.abs().amax(-1).clamp(min=1e-30) / 448.0
    return (x / scale.unsqueeze(-1)).to(torch.float8_e4m3fn), scale


def values64(pages, scale):
    x = pages.to(torch.float32).double().numpy()
    return x if scale is None else x * scale.double().numpy()[..., None]


def tables(lengths, page, num_pages, rng, extra=0, fill=-1):
    """Every sequence's own pages in random order, `extra` more entries of `fill` at the end."""
    per = max([-(-n // page) for n in lengths] + [0]) + extra
    order = rng.permutation(num_pages)
    t = np.full((len(lengths), per), fill, np.int32)
    used = 0
    for s, n in enumerate(lengths):
        k = -(-n // page)
        t[s, :k] = order[used:used + k]
        used += k
    return t


def slots_of(table, n, page, num_pages):
    """(slot numbers t, page, row) of a sequence's present slots."""
    t = np.arange(n)
    p = table[t // page] if n else np.zeros(0, np.int64)
    there = (p >= 0) & (p < num_pages)
    return t[there], p[there].astype(np.int64), (t % page)[there]


def attend(q, k64, v64, table, lengths, scale, dtype, cache):
    """out, lse, added weights [P, H, page] and the bounds on each one's error.

    The kernel multiplies in the inputs' type and adds in f32 (D products: at most
    D * 2^-24 of the sum of their magnitudes), takes exp2 of a score times log2(e)
    (a few 2^-24, and 2^-24 of the score's size), keeps at least 16 bits of a
    weight that enters the product with 16- or 8-bit values, and rounds once."""
    S, Hq, D = q.shape
    P, H, page, _ = k64.shape
    q64 = q.to(torch.float32).double().numpy()
    out, lse, added = np.zeros((S, Hq, D)), np.full((S, Hq), -math.inf), np.zeros((P, H, page))
    b_out, b_lse, b_added = np.zeros((S, Hq, D)), np.zeros((S, Hq)), np.zeros((P, H, page))
    kept = 0.0 if cache == "f32" else 2.0**-16
    for s in range(S):
        _, p, o = slots_of(table[s], int(lengths[s]), page, P)
        if p.size == 0:
            continue
        for h in range(Hq):
            g = h // (Hq // H)
            k, v = k64[p, g, o], v64[p, g, o]
            with np.errstate(invalid="ignore"):
                x = scale * (k @ q64[s, h])
            size = abs(scale) * (np.abs(k) @ np.abs(q64[s, h])).max() if np.isfinite(x).all() else 0.0
            top = x.max()
            if top == -math.inf:
                continue
            e = np.exp(x - top)
            w = e / e.sum()
            rel = 2 * (D + 8) * 2.0**-24 * size + 2.0**-20  # of a weight: scores, exp2, the sum
            rel += 2.0**-23 * math.log2(p.size + 1)
            out[s, h] = w @ v
            lse[s, h] = top + math.log(e.sum())
            mass = w @ np.abs(v)
            b_out[s, h] = (rel + kept) * mass * 1.01 + HALF_ULP[dtype] * np.maximum(
                np.abs(out[s, h]) + (rel + kept) * mass, SMALL[dtype])
            b_lse[s, h] = rel + 2.0**-22 * abs(lse[s, h])
            added[p, g, o] += w
            b_added[p, g, o] += 2 * rel * w + 2.0**-24 * w * (Hq // H)
    return out, lse, added, b_out, b_lse, b_added


def rotate(x, positions, cos_sin, sections, interleaved):
    """x [T, heads, D] of any type, rotated in f32 (two products, one sum, each rounded)."""
    x = x.to(torch.float32).numpy().copy()
    if cos_sin is None:
        return x
    rot, half = cos_sin.shape[1], cos_sin.shape[1] // 2
    positions = positions if positions.ndim == 2 else positions[None]
    axis = np.repeat(np.arange(len(sections)), sections)
    for i in range(half):
        p = positions[axis[i]]
        there = (p >= 0) & (p < cos_sin.shape[0])
        c = cos_sin[np.where(there, p, 0), i][:, None]
        s = cos_sin[np.where(there, p, 0), half + i][:, None]
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        xa, xb = x[:, :, a].copy(), x[:, :, b].copy()
        x[:, :, a] = np.where(there[:, None], xa * c - xb * s, xa)
        x[:, :, b] = np.where(there[:, None], xb * c + xa * s, xb)
    return x


def quantize(x):
    """f32 rows to e4m3 codes (as torch.float8_e4m3fn) and scales."""
    x = torch.from_numpy(x)
    scale = x.abs().amax(-1).clamp(min=np.float32(1e-30)) / np.float32(448.0)
    return (x / scale.unsqueeze(-1)).to(torch.float8_e4m3fn), scale


def evict(weights, index, table, lengths, budget, sinks, recent, page):
    """The moves (head, to (page, row), from (page, row)) of every sequence, in order, and the new lengths."""
    P, H, _ = weights.shape
    moves, new = [], []
    for s, n in enumerate(lengths):
        n = min(max(int(n), 0), table.shape[1] * page)
        keep = min(n, budget)
        new.append(keep)
        if keep == n or keep == 0:
            continue
        for h in range(H):
            def where(t):
                p = int(table[s, t // page])
                return (p, t % page) if 0 <= p < P else None

            at = [where(t) for t in range(n)]
            newest = max([int(index[a[0], h, a[1]]) for a in at if a] + [-(1 << 62)])

            def rank(t):
                if at[t] is None:
                    return (0, 0, 0.0, t)
                i, w = int(index[at[t][0], h, at[t][1]]), float(weights[at[t][0], h, at[t][1]])
                held = 1 if i < sinks or i > newest - recent else 0
                return (held, 1, math.inf, t + (1 << 40)) if w != w else (held, 1, w, t)

            order = sorted(range(n), key=rank)
            dropped = set(order[:n - keep])
            holes = [t for t in range(keep) if t in dropped]
            movers = [t for t in range(keep, n) if t not in dropped]
            assert len(holes) == len(movers)
            moves += [(h, at[a], at[b]) for a, b in zip(holes, movers) if at[a] and at[b]]
    return moves, new
