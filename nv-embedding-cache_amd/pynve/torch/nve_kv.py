"""The paged key-value cache of an attention layer, for models that answer one token at a time.

A model that reads its token or item embeddings through the lookup layers and
answers step by step keeps the keys and values of what it has seen.  Here they
lie in pages of a few slots; a sequence is a row of page numbers.  Three
operators work on the pages, each one a hand-written HIP kernel behind the C ABI
(nve_amd_kv_*) and a torch op (torch.ops.nve_ops.kv_*):

  kv_append   rotary positions on new queries and keys, keys and values into their slots
  kv_attend   attention of one new token per sequence over its pages; can add each slot's attention
              weight to the weight the cache holds for it
  kv_evict    drops the slots of the least accumulated weight from sequences that are over a budget

`KVCache` holds the pages and calls the three.  Everything runs on the current
stream of the pages' GPU, nothing waits for the GPU, and nothing has a gradient:
inputs that ask for one are refused unless gradients are off.

Shapes (P pages, H key heads, `page` slots a page, D values a head row, S sequences, T tokens):

  k_pages, v_pages   [P, H, page, D]  float32, float16, bfloat16 or float8_e4m3fn
  k_scale, v_scale   [P, H, page]     float32, float8 pages only: a row's value is code * scale
  weights            [P, H, page]     float32, accumulated attention weight
  index_pages        [P, H, page]     int32, the token's place in its sequence
  block_tables       [S, pages]       int32; slot t of sequence s is row t % page of page
                                      block_tables[s, t // page]
  lengths            [S]              int32

`page` is a power of two from 8 to 1024, D a multiple of 8 up to 256.  Page
numbers outside [0, P) name no page: their slots are neither read nor written.
"""
import torch

from . import HAS_TORCH_OPS  # noqa: F401  (importing registers the ops)

_append = torch.ops.nve_ops.kv_append.default
_attend = torch.ops.nve_ops.kv_attend.default
_attend_lse = torch.ops.nve_ops.kv_attend_lse.default
_evict = torch.ops.nve_ops.kv_evict.default


def kv_append(k, v, k_pages, v_pages, slots, *, q=None, positions=None, cos_sin=None, sections=None,
              interleaved=False, index=None, k_scale=None, v_scale=None, weights=None, index_pages=None):
    """Writes the keys and values of T new tokens [T, H, D] to the slots `slots`
    (int64: page number * page + row; a slot outside the cache is skipped, none
    may appear twice) and returns the rotated queries, or None without `q`.

    With `cos_sin` (float32 [positions, R]: the cosines of R / 2 pairs, then
    their sines) the first R values of every query and key head are rotated by
    `positions` (int32 [T], or [axes, T] for up to four axes such as time, height
    and width).  Pair i is values i and i + R / 2, or 2i and 2i + 1 if
    `interleaved`; the first sections[0] pairs turn by axis 0, the next
    sections[1] by axis 1 and so on.  A position outside the table leaves its
    pairs as they are.  `index` (int32 [T], by default positions of axis 0, or 0)
    goes to index_pages, 0 to weights.  Strides are free but for the last
    dimension."""
    out = _append(k, v, k_pages, v_pages, slots, q, positions, cos_sin, sections, interleaved, index, k_scale,
                  v_scale, weights, index_pages)
    return None if q is None else out


def kv_attend(q, k_pages, v_pages, block_tables, lengths, *, scale=None, k_scale=None, v_scale=None, weights=None,
              max_length=None, return_lse=False):
    """Attention of one query token per sequence, q [S, Hq, D], over its slots
    t < lengths[s]: softmax(scale * q . k) v, query head h on key head
    h // (Hq // H); `scale` is 1 / sqrt(D) by default.  Returns [S, Hq, D] of q's
    type, with `return_lse` also the logarithm of each softmax's sum, float32
    [S, Hq].  A sequence without slots gives zeros (and -inf).  With `weights` the
    softmax of every slot, summed over the query heads of its key head, is added
    there; no page may then belong to two of the sequences.  Sums are float32; the
    softmax values that meet float16 values keep 22 bits, those that meet float8
    values 17.  `max_length` is a bound on the lengths if the caller knows one below
    the tables' extent; it sizes the launch and the workspace."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    f = _attend_lse if return_lse else _attend
    return f(q, k_pages, v_pages, block_tables, lengths, scale, k_scale, v_scale, weights, max_length or 0)


def kv_evict(k_pages, v_pages, weights, index_pages, block_tables, lengths, budget, *, sinks=0, recent=0,
             k_scale=None, v_scale=None):
    """Brings every sequence of more than `budget` slots down to `budget` and
    returns the new lengths.  Each key head drops the slots lowest in (protected,
    weight, slot); protected are a head's slots with an index below `sinks` and
    those among the `recent` places up to its newest index.  Kept slots past the
    budget move into the gaps below it, so the order of the slots changes
    (attention does not depend on it; index_pages says which token a slot holds).
    Pages past ceil(new length / page) are free for other sequences.  A row whose
    gap lies in an absent page is lost: absent pages belong behind a table's others."""
    return _evict(k_pages, v_pages, weights, index_pages, block_tables, lengths, budget, sinks, recent, k_scale,
                  v_scale)


class KVCache:
    """Pages of one attention layer and their companions.

    `dtype` is that of the queries and keys, or torch.float8_e4m3fn (with
    float16 or bfloat16 queries); `track_weights=False` leaves out what eviction
    needs (weights and index)."""

    def __init__(self, num_pages, num_kv_heads, head_dim, page=16, dtype=torch.float16, device="cuda",
                 track_weights=True):
        shape = (num_pages, num_kv_heads, page)
        self.page = page
        self.k = torch.zeros((*shape, head_dim), dtype=dtype, device=device)
        self.v = torch.zeros((*shape, head_dim), dtype=dtype, device=device)
        scaled = dtype == torch.float8_e4m3fn
        self.k_scale = torch.zeros(shape, dtype=torch.float32, device=device) if scaled else None
        self.v_scale = torch.zeros(shape, dtype=torch.float32, device=device) if scaled else None
        self.weights = torch.zeros(shape, dtype=torch.float32, device=device) if track_weights else None
        self.index = torch.zeros(shape, dtype=torch.int32, device=device) if track_weights else None

    def slots(self, block_tables, seq, place):
        """The slot numbers of places `place` in sequences `seq` (int64 tensors of one shape)."""
        return block_tables[seq, place // self.page].long() * self.page + place % self.page

    def append(self, k, v, slots, *, q=None, positions=None, cos_sin=None, sections=None, interleaved=False,
               index=None):
        """kv_append on these pages."""
        return kv_append(k, v, self.k, self.v, slots, q=q, positions=positions, cos_sin=cos_sin, sections=sections,
                         interleaved=interleaved, index=index, k_scale=self.k_scale, v_scale=self.v_scale,
                         weights=self.weights, index_pages=self.index)

    def attend(self, q, block_tables, lengths, *, scale=None, accumulate=None, max_length=None, return_lse=False):
        """kv_attend on these pages; accumulates weights where the cache tracks them, unless told not to."""
        if accumulate is None:
            accumulate = self.weights is not None
        if accumulate and self.weights is None:
            raise ValueError("accumulate: this cache was made with track_weights=False")
        return kv_attend(q, self.k, self.v, block_tables, lengths, scale=scale, k_scale=self.k_scale,
                         v_scale=self.v_scale, weights=self.weights if accumulate else None, max_length=max_length,
                         return_lse=return_lse)

    def evict(self, block_tables, lengths, budget, *, sinks=0, recent=0):
        """kv_evict on these pages."""
        if self.weights is None:
            raise ValueError("evict: this cache was made with track_weights=False")
        return kv_evict(self.k, self.v, self.weights, self.index, block_tables, lengths, budget, sinks=sinks,
                        recent=recent, k_scale=self.k_scale, v_scale=self.v_scale)


@torch.library.register_fake("nve_ops::kv_append")
def _kv_append_fake(k, v, k_pages, v_pages, slots, q, *rest):
    return k.new_empty((0,) if q is None else q.shape)


@torch.library.register_fake("nve_ops::kv_attend")
def _kv_attend_fake(q, *rest):
    return q.new_empty(q.shape)


@torch.library.register_fake("nve_ops::kv_attend_lse")
def _kv_attend_lse_fake(q, *rest):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


@torch.library.register_fake("nve_ops::kv_evict")
def _kv_evict_fake(k_pages, v_pages, weights, index_pages, block_tables, lengths, *rest):
    return lengths.new_empty(lengths.shape)
