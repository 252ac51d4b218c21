"""Plain 64-bit forms of the rotation, the cache's append and the attention of packed sequences (not collected)."""
import math

import torch


def half_step(dtype):
    """What a rounding to ``dtype`` is off by at most, relative to the value."""
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """... and below the smallest normal number, as a value."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def norm_rotate(x, w, angles, eps, interleaved):
    """x [..., D] (any dtype), angles [..., rot] = cosines, sines: the result in 64 bits, and the sum of the magnitudes
    that an element is made of."""
    x = x.double()
    rot = angles.shape[-1]
    cos, sin = angles[..., :rot // 2].double(), angles[..., rot // 2:].double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    ya, yb = a * cos - b * sin, b * cos + a * sin
    ma, mb = (a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()
    join = (lambda s, t: torch.stack([s, t], -1).flatten(-2)) if interleaved else (lambda s, t: torch.cat([s, t], -1))
    return torch.cat([join(ya, yb), x[..., rot:]], -1), torch.cat([join(ma, mb), x[..., rot:].abs()], -1)


def rotate_bound(y, magnitude, dtype):
    """One rounding of the result; before it a dozen 32-bit operations on its terms (the mean of up to 256 squares, added
    up by a tree of 8 levels and chains of 16, a root and a quotient among them): 2^-24 each, 40 of them."""
    return half_step(dtype) * y.abs() * (1 + 1e-3) + 40 * 2.0 ** -24 * magnitude + smallest(dtype)


def attention(q, k, v, first, causal, softcap):
    """q [n, Hq, D] (row i at position first + i), k, v [m, Hk, D]: o, the weighted mean of |v|, lse, in 64 bits.
    Only allowed keys are ever multiplied by anything."""
    n, Hq, D = q.shape
    m, Hk = k.shape[0], k.shape[1]
    G = Hq // Hk
    o = torch.zeros(n, Hq, D, dtype=torch.float64, device=q.device)
    mean = torch.zeros_like(o)
    lse = torch.full((n, Hq), -math.inf, dtype=torch.float64, device=q.device)
    for h in range(Hq):
        kh, vh = k[:, h // G].double(), v[:, h // G].double()
        x = (q[:, h].double() @ kh.t()) / math.sqrt(D)
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        allowed = torch.ones(n, m, dtype=torch.bool, device=q.device)
        if causal:
            allowed = torch.arange(m, device=q.device) <= first + torch.arange(n, device=q.device).unsqueeze(1)
        x = torch.where(allowed, x, torch.full_like(x, -math.inf))
        lse[:, h] = torch.logsumexp(x, -1) if m else lse[:, h]
        live = allowed.any(-1) if m else torch.zeros(n, dtype=torch.bool, device=q.device)
        if not bool(live.any()):
            continue
        p = torch.softmax(x[live], -1)
        if bool(torch.isfinite(vh).all()):
            o[live, h], mean[live, h] = p @ vh, p @ vh.abs()
        else:
            terms = torch.where(allowed[live].unsqueeze(-1), p.unsqueeze(-1) * vh, torch.zeros((), dtype=torch.float64, device=q.device))
            o[live, h], mean[live, h] = terms.sum(1), terms.abs().sum(1)
    return o, mean, lse


def attention_bound(o, mean, vmax, dtype, softcap, D, smax):
    """Weights are rounded to 16 bits before the second product and the result once more: half a step of the weighted
    mean of |v|, half a step of the result.  Weights of less than the smallest normal number of fp16 are off by half its
    smallest step each, against sums of at least 2^-7 (a row's reference lies at most 2^6 above its first maximum, and
    that within 1): with vmax the largest |v| times the keys.  Before that 32 bits: a score of D products, at most smax,
    is off by D 2^-24 smax, a capped one by a few steps of the cap, exponent and exponential by as much again, and a
    weight by that relative to itself."""
    scores = (D * 2.0 ** -24 + 4 * 2.0 ** -23) * smax + 8 * 2.0 ** -23 * softcap + 8 * 2.0 ** -23
    weights = half_step(dtype) * (1 + 1e-3) + 2 * scores
    tiny = smallest(dtype) * 128 * vmax if dtype == torch.float16 else 0.0
    return weights * mean + half_step(dtype) * o.abs() + smallest(dtype) + tiny


def offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out
