"""Token sampling: the last operator of a model's step, beside the key-value cache's (nve_kv).

`sample_tokens` draws a token for every row of logits from one random number
of the caller's, after temperature, top-k, top-p and min-p, in hand-written HIP
kernels behind the C ABI (nve_amd_sample) and a torch op
(torch.ops.nve_ops.sample_tokens).  It runs on the current stream of the
logits' GPU, does not wait for the GPU, can be captured into a graph and has no
gradient: logits that ask for one are refused unless gradients are off.
"""
import torch

from . import HAS_TORCH_OPS  # noqa: F401  (importing registers the ops)

_sample = torch.ops.nve_ops.sample_tokens.default


def sample_tokens(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token for every row of `logits` [rows, vocabulary] (float32, float16 or
    bfloat16, the rows at any stride), drawn with `u` (float32 [rows], uniform in
    [0, 1)); int64 [rows].

    With w = exp((logits - their maximum) / temperature) a token is kept if it is
    among the `top_k` first (0: all) in the order (logit descending, index
    ascending), if the sum before it in that order is below `top_p` times the sum
    over those (1 or more: all; the first token is always kept), and if w >=
    `min_p`.  The token is the first index, in the vocabulary's order, at which the
    running sum of the kept w exceeds u times their sum.  A temperature of 0 takes
    the first of the largest logits.  Exponentials and sums are 64-bit; in the sum over
    a whole row of 16-bit logits a weight is within 2^-31 of its value.

    Each limit is a number or a tensor [rows] (float32; top_k int32) on the logits'
    GPU, where a temperature that is not above 0 counts as 0, a top_k below 1 as 0 and
    a top_p or min_p that is no number as none.  Logits that are no number count as
    minus infinity; a row of nothing else gives -1.  Where a logit is plus infinity
    only such logits have a weight.

    Made for vocabularies up to 2^19 and a top_k up to about 2,000: past these (up to
    2^30) a row is one workgroup's, 5 to 40 times slower."""
    limits = {"temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p}
    each = [x if isinstance(x, torch.Tensor) else None for x in limits.values()]
    every = [0 if isinstance(x, torch.Tensor) else x for x in limits.values()]
    return _sample(logits, u, *each, *every)


@torch.library.register_fake("nve_ops::sample_tokens")
def _sample_tokens_fake(logits, u, *rest):
    return logits.new_empty((logits.shape[0],), dtype=torch.int64)
