"""The operators together, as a model is served: prompts go through the rotation and the packed attention and into the cache,
then tokens one by one; every step against the whole sequences at once.  And a training step of a layer: norms, rotation and
the block-sparse attention."""
import pytest
import torch

import omni_attn_torch as oat
from serving_helpers import attention, norm_rotate, offsets

pytestmark = pytest.mark.gpu

EPS = 1e-5


@pytest.mark.parametrize("dtype,Hq,Hk,D,page", [(torch.bfloat16, 8, 2, 128, 32), (torch.float16, 4, 4, 64, 16)])
def test_prompts_then_tokens(gpu_device, dtype, Hq, Hk, D, page):
    gen = torch.Generator().manual_seed(1)
    prompts, steps = [37, 1, 130], 5
    B = len(prompts)
    total = [n + steps for n in prompts]
    make = lambda n, H: torch.randn(n, H, D, generator=gen).to(device=gpu_device, dtype=dtype)
    q, k, v = ([make(n, H) for n in total] for H in (Hq, Hk, Hk))
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=gen)).to(device=gpu_device, dtype=dtype) for _ in range(2))
    table = oat.omni_rotary_table(D, max(total), device=gpu_device)
    need = [-(-n // page) for n in total]
    kp, vp = (torch.full((sum(need), Hk, page, D), float("nan"), dtype=dtype, device=gpu_device) for _ in range(2))
    pages = torch.zeros(B, max(need), dtype=torch.int32)
    for b, order in enumerate(torch.randperm(sum(need), generator=gen).to(torch.int32).split(need)):
        pages[b, :need[b]] = order
    pages = pages.to(gpu_device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    outs = [[] for _ in range(B)]

    # the prompts: rotated packed, attended packed, and appended
    at = offsets(prompts)
    pq, pk, pv = (torch.cat([x[b][:n] for b, n in enumerate(prompts)]) for x in (q, k, v))
    positions = torch.cat([torch.arange(n) for n in prompts]).to(gpu_device)
    rq, rk = oat.omni_qk_rotary(pq, pk, positions, table, wq, wk, EPS)
    o = oat.omni_attention_packed(rq, rk, pv, i32(at))
    aq = oat.omni_cache_append(pk, pv, kp, vp, pages, i32(prompts), i32(at), table=table, query=pq, query_norm=wq, key_norm=wk, eps=EPS)
    assert torch.equal(aq, rq)  # the same arithmetic
    again = oat.omni_attention_paged(aq, kp, vp, pages, i32(prompts), i32(at))
    assert (again.float() - o.float()).abs().max().item() <= 8 * torch.finfo(dtype).eps
    for b in range(B):
        outs[b].append(o[at[b]:at[b + 1]])
    # tokens
    for s in range(steps):
        tq, tk, tv = (torch.stack([x[b][prompts[b] + s] for b in range(B)]) for x in (q, k, v))
        kv = i32([n + s + 1 for n in prompts])
        cu = i32(list(range(B + 1)))
        y = oat.omni_cache_append(tk, tv, kp, vp, pages, kv, cu, table=table, query=tq, query_norm=wq, key_norm=wk, eps=EPS)
        o = oat.omni_attention_paged(y, kp, vp, pages, kv, cu)
        for b in range(B):
            outs[b].append(o[b:b + 1])
    for b in range(B):
        angles = table[:total[b]].unsqueeze(1)
        rq, rk = norm_rotate(q[b], wq, angles, EPS, False)[0], norm_rotate(k[b], wk, angles, EPS, False)[0]
        want, mean, _ = attention(rq, rk, v[b], 0, True, 0.0)
        # rotated heads are rounded (half a step each, so scores of |q| |k| / sqrt(D) are off by two half steps and weights by
        # e to that), weights once more, results once more
        eps = torch.finfo(dtype).eps / 2
        smax = (rq.norm(dim=-1).max() * rk.norm(dim=-1).max()).item() / D ** 0.5
        bound = mean * (2 * (2 * eps * smax) + 2 * eps) + eps * want.abs() + 1e-6
        assert bool(((torch.cat(outs[b]).double() - want).abs() <= bound).all()), b


def test_a_training_layer(gpu_device):
    """Gradients of the block-sparse attention go on through rotation and norm: against 64 bits."""
    gen = torch.Generator().manual_seed(2)
    dtype, B, S, H, D = torch.float16, 2, 256, 2, 64
    x = [(torch.randn(B, S, H, D, generator=gen)).to(device=gpu_device, dtype=dtype).requires_grad_() for _ in range(3)]
    w = [(1 + 0.2 * torch.randn(D, generator=gen)).to(device=gpu_device, dtype=dtype).requires_grad_() for _ in range(2)]
    table = oat.omni_rotary_table(D, S, device=gpu_device)
    positions = torch.arange(S, device=gpu_device)
    q, k, v = (t.transpose(1, 2) for t in x)
    mask = oat.create_causal_omni_block_mask(B, H, S, S, device=gpu_device)
    rq, rk = oat.omni_qk_rotary(q, k, positions, table, w[0], w[1], EPS)
    o = oat.omni_attention(rq, rk, v, mask)
    do = torch.randn(o.shape, generator=gen).to(device=gpu_device, dtype=dtype)
    grads = torch.autograd.grad(o, x + w, do)
    wx = [t.detach().double().requires_grad_() for t in x]
    ww = [t.detach().double().requires_grad_() for t in w]
    rq = norm_rotate(wx[0].transpose(1, 2), ww[0], table, EPS, False)[0]
    rk = norm_rotate(wx[1].transpose(1, 2), ww[1], table, EPS, False)[0]
    scores = (rq @ rk.transpose(-1, -2)) / D ** 0.5
    scores = scores.masked_fill(torch.ones(S, S, dtype=torch.bool, device=gpu_device).triu(1), float("-inf"))
    ref = torch.softmax(scores, -1) @ wx[2].transpose(1, 2)
    want = torch.autograd.grad(ref, wx + ww, do.double())
    for i, (a, b) in enumerate(zip(grads, want)):
        assert bool(torch.isfinite(a.float()).all())
        # the operator's own gradients are within 2e-2 of theirs; the rotation adds a rounding
        assert (a.double() - b).abs().max().item() <= 2e-2 * b.abs().max().item(), i
