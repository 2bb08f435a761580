"""The draw of the next token on the HIP engine (the sampling steps of models/lm.py:138-143, with the random numbers
given and top-p and min-p beside top-k)."""

from . import _abi


def sample(logits, u, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """(token, logprob) of every row of logits (..., V), V <= 2^24, float32, bfloat16 or float16.

    With w_i = exp((l_i - max l) / temperature): of the order by falling logit (ties: the lower index first) the first
    top_k are kept, of those the shortest prefix with top_p of their mass, of those the ones with w_i >= min_p, and
    always the first.  token (...) int64 is the first kept index at which the running sum of the kept w, by index,
    passes u times their sum; logprob (...) float32 the log of its share of that sum.

    u (...) float32 or float64 in [0, 1), as torch.rand gives it.  Each setting is a number or a tensor with one per
    row, read in float32 (top_k in int64): temperature 0 takes the first of the order; top_k None or 0, top_p None or 1,
    min_p None or 0 keep all.  In a tensor, a temperature below 0 or NaN counts as 0, a top_k below 0 as 0.  A row with a
    NaN, or with no logit above -inf, gives token -1 and logprob NaN.  Not differentiable: in grad mode, logits that
    require a gradient are refused.

    Weights are rounded to 2^-S of the largest, S = min(51, 62 - the bits of V), and their sums are exact, so the same
    inputs give the same tokens.  V of them may lose V 2^-(S+1) of the largest: 4e-9 at V = 131072, 2.4e-7 at 2^20, 6e-5
    at 2^24; one below 2^-(S+1) is not drawn."""
    return _abi.host().sample(logits, u, temperature, top_k, top_p, min_p)
