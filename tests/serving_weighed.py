"""Batches whose parts are weighed on the device, and how far off the attention over a cache may be (not collected)."""
import math

import torch

from serving_helpers import half_step, smallest

# (new tokens, keys before them, query heads, key heads, head_dim): single tokens and a few, then chunks of prompts
FEW = [
    ([1], [60000], 32, 8, 128), ([1] * 4, [1000, 3300, 8000, 5100], 32, 8, 128), ([1] * 8, [300, 16000, 700, 9000, 5, 2500, 64, 12345], 16, 8, 64),
    ([2, 0, 1, 0, 3], [9000, 40, 12000, 0, 5000], 16, 8, 32), ([1], [40000], 4, 2, 128), ([3, 1], [11000, 9000], 4, 4, 64),
    ([1, 1, 1], [0, 39999, 20000], 3, 3, 32),
]
CHUNKS = [
    ([100], [20000], 8, 1, 128), ([512, 300], [3000, 1401], 8, 2, 64), ([40, 300, 7, 0, 200], [6000, 9000, 2500, 900, 7000], 3, 1, 32),
    ([33] * 16, [1000 + 700 * b for b in range(16)], 8, 1, 64), ([200, 0, 130], [9000, 700, 11000], 8, 2, 128),
]


def reference(q, k, v, first, causal):
    """q [n, Hq, D] (row i at position first + i), k, v [m, Hk, D]: o, the weighted mean of |v|, the logsumexp and what an
    absolute error of one in every weight, against the row's maximum, would come to in o; in 64 bits."""
    n, Hq, D = q.shape
    m, G = k.shape[0], Hq // k.shape[1]
    o, mean, spread = (torch.zeros(n, Hq, D, dtype=torch.float64, device=q.device) for _ in range(3))
    lse = torch.full((n, Hq), -math.inf, dtype=torch.float64, device=q.device)
    live = torch.arange(n, device=q.device) + first >= 0 if causal else torch.ones(n, dtype=torch.bool, device=q.device)
    if m == 0 or not bool(live.any()):
        return o, mean, lse, spread
    allowed = torch.ones(n, m, dtype=torch.bool, device=q.device)
    if causal:
        allowed = torch.arange(m, device=q.device) <= first + torch.arange(n, device=q.device).unsqueeze(1)
    for h in range(Hq):
        kh, vh = k[:, h // G].double(), v[:, h // G].double()
        x = ((q[:, h].double() @ kh.t()) / math.sqrt(D)).masked_fill(~allowed, -math.inf)[live]
        top = x.amax(-1, keepdim=True)
        w = torch.exp(x - top)
        total = w.sum(-1, keepdim=True)
        lse[live, h] = (top + total.log()).squeeze(-1)
        o[live, h], mean[live, h] = w @ vh / total, w @ vh.abs() / total
        spread[live, h] = allowed[live].double() @ vh.abs() / total
    return o, mean, lse, spread


def bound(o, mean, spread, dtype, D, smax):
    """A weight is rounded to 16 bits once (half a step of it), and so is the result.  An fp16 weight below the smallest
    normal number is off by half its smallest step against the row's reference, which is a maximum of scores of the row's own
    keys and so at most the row's maximum: the sum of weights against the reference is at least that against the maximum,
    and where parts are joined, weights of lower references are scaled down, their errors with them.  32 bits before that: a
    score of D products of at most smax in all is off by D 2^-24 smax and its scaling and the reference's by a few steps, a
    weight by as much relative to itself, and the sum below it too."""
    scores = (D * 2.0 ** -24 + 4 * 2.0 ** -23) * smax + 8 * 2.0 ** -23
    weights = half_step(dtype) * (1 + 1e-3) + 2 * scores
    tiny = smallest(dtype) * (1 + 1e-3) * spread if dtype == torch.float16 else 0.0
    return weights * mean + half_step(dtype) * o.abs() + smallest(dtype) + tiny


def make(gen, lens, cached, Hq, Hk, D, dtype, behind=0):
    """Queries of all tokens, and keys and values per sequence.  Values rise or fall along a sequence, so that a key left out
    or counted twice shows in every sum."""
    q = torch.randn(sum(lens) + behind, Hq, D, generator=gen).to(dtype)
    rows = []
    for n, c in zip(lens, cached):
        m = n + c
        slope = (torch.arange(D) % 5 - 2.0) * 1.5
        ramp = torch.arange(m).view(m, 1, 1) / max(m, 1) * slope
        rows.append((torch.randn(m, Hk, D, generator=gen).to(dtype), (torch.randn(m, Hk, D, generator=gen) + ramp + 0.5).to(dtype)))
    return q, rows
