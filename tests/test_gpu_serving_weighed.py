"""Parts that are weighed on the device, over a paged cache: single tokens, a few and chunks of prompts of up to 16 sequences,
against 64 bits."""
import math

import pytest
import torch

import omni_attn_torch as oat
from serving_helpers import offsets
from serving_weighed import CHUNKS, FEW, bound, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", range(len(FEW) + len(CHUNKS)))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [32, 64])
def test_weighed_parts(gpu_device, case, dtype, page):
    lens, cached, Hq, Hk, D = (FEW + CHUNKS)[case]
    gen = torch.Generator().manual_seed(case)
    q, rows = make(gen, lens, cached, Hq, Hk, D, dtype, behind=3)
    q, rows = q.to(gpu_device), [(k.to(gpu_device), v.to(gpu_device)) for k, v in rows]
    total = [n + c for n, c in zip(lens, cached)]
    need = [-(-n // page) for n in total]
    order = torch.randperm(sum(need) + 2, generator=gen)
    pools = [torch.full((sum(need) + 2, Hk, page, D), float("nan"), dtype=dtype, device=gpu_device) for _ in range(2)]
    table, at = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        own = order[at:at + n]
        table[b, :n] = own.to(torch.int32)
        at += n
        for pool, x in zip(pools, rows[b]):
            wide = torch.full((n * page, Hk, D), float("nan"), dtype=dtype, device=gpu_device)
            wide[:total[b]] = x
            pool[own.to(gpu_device)] = wide.view(n, page, Hk, D).transpose(1, 2)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    cu = offsets(lens)
    for causal in (True, False):
        o, lse = oat.omni_attention_paged(q, *pools, table.to(gpu_device), i32(total), i32(cu), causal=causal, return_lse=True)
        assert bool((o[cu[-1]:] == 0).all()) and bool((lse[cu[-1]:] == -math.inf).all())
        for b, (k, v) in enumerate(rows):
            a, e = cu[b], cu[b + 1]
            if a == e:
                continue
            want, mean, rl, spread = reference(q[a:e], k, v, cached[b], causal)
            smax = (q[a:e].double().norm(dim=-1).max() * k.double().norm(dim=-1).max()).item() / math.sqrt(D)
            over = (o[a:e].double() - want).abs() - bound(want, mean, spread, dtype, D, smax)
            assert bool((over <= 0).all()), f"sequence {b}: beyond its bound by {over.max().item():.3e}"
            room = (D + 8) * 2.0 ** -24 * smax + 2.0 ** -21 * (1 + rl.abs())
            assert bool(((lse[a:e].double() - rl).abs() <= room).all()), b
        assert torch.equal(oat.omni_attention_paged(q, *pools, table.to(gpu_device), i32(total), i32(cu), causal=causal), o)
