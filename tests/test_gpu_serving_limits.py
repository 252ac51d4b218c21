"""Calls of the packed-sequence operators at their limits: offsets that run backwards, values that are no numbers, scratch memory."""
import pytest
import torch

import omni_attn_torch as oat
from serving_helpers import attention, attention_bound, offsets

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [65, 130, 700])
@pytest.mark.parametrize("D", [32, 128])
def test_backward_offsets_of_many_sequences(gpu_device, B, D):
    """More than 64 sequences, some of them empty between offsets that run backwards, at the buffers' ends too: every call ends."""
    gen = torch.Generator().manual_seed(B + D)
    dtype, T, Hq, Hk, page = torch.bfloat16, 600, 4, 1, 16
    q, k, v, do = (torch.randn(T, h, D, generator=gen).to(device=gpu_device, dtype=dtype) for h in (Hq, Hk, Hk, Hq))
    kp, vp = (torch.randn(200, Hk, page, D, generator=gen).to(device=gpu_device, dtype=dtype) for _ in range(2))
    table = torch.randint(0, 200, (B, 90), generator=gen).to(device=gpu_device, dtype=torch.int32)
    for case in range(4):
        cu = torch.randint(0, T + 1, (B + 1,), generator=gen)
        cu[torch.rand(B + 1, generator=gen) < (0.8 if case % 2 else 0.3)] = T if case < 2 else 0
        cu = cu.to(device=gpu_device, dtype=torch.int32)
        kv = torch.randint(0, 90 * page, (B,), generator=gen).to(device=gpu_device, dtype=torch.int32)
        for causal in (True, False):
            leaves = [t.detach().requires_grad_() for t in (q, k, v)]
            o = oat.omni_attention_packed(*leaves, cu, causal=causal)
            grads = torch.autograd.grad(o, leaves, do)
            p = oat.omni_attention_paged(q, kp, vp, table, kv, cu, causal=causal)
            torch.cuda.synchronize()
            assert p.shape == o.shape and [g.shape for g in grads] == [t.shape for t in leaves]
    # and a batch whose offsets do not decrease is right after them
    cu = torch.linspace(0, T, B + 1).to(torch.int32).to(gpu_device)
    a, b = int(cu[B // 2]), int(cu[B // 2 + 1])
    one = torch.tensor([0, b - a], dtype=torch.int32, device=gpu_device)
    if b > a:
        got = oat.omni_attention_packed(q, k, v, cu)[a:b].float()
        want = oat.omni_attention_packed(q[a:b].contiguous(), k[a:b].contiguous(), v[a:b].contiguous(), one).float()
        # two roundings of weights and results each, of values of at most 5
        assert (got - want).abs().max().item() <= 4 * 5 * torch.finfo(dtype).eps / 2


def _paged_of(gen, k, v, lens, page):
    """Packed keys and values in pages of a shuffled cache: key_pages, value_pages, page_table."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + 2, generator=gen)
    pools = [torch.full((sum(need) + 2, k.shape[1], page, k.shape[2]), float("nan"), dtype=k.dtype, device=k.device) for _ in range(2)]
    table, at, row = torch.zeros(len(lens), max(need), dtype=torch.int32), 0, 0
    for b, n in enumerate(lens):
        own = order[at:at + need[b]]
        table[b, :need[b]] = own.to(torch.int32)
        at += need[b]
        for pool, x in zip(pools, (k, v)):
            for i, pg in enumerate(own.tolist()):
                part = x[row + i * page:row + min(n, (i + 1) * page)]
                pool[pg, :, :part.shape[0]] = part.transpose(0, 1)
        row += n
    return pools[0], pools[1], table.to(k.device)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Hq,Hk,D,lens,softcap", [
    (4, 4, 64, [200], 0.0), (8, 2, 128, [130, 77], 0.0), (8, 1, 32, [300, 5], 20.0),  # few rows, four waves
    (16, 16, 128, [1300], 0.0), (16, 16, 64, [700, 90], 15.0),                        # tiles of 64 rows
    (32, 8, 128, [1500, 300], 0.0), (24, 24, 32, [1600], 0.0),                        # of 128, whole
    (8, 8, 64, [70] * 40, 0.0)])                                                      # few rows, one wave
@pytest.mark.parametrize("page", [0, 16, 64])
def test_no_numbers_by_right_and_behind_a_row(gpu_device, dtype, Hq, Hk, D, lens, softcap, page):
    """Infinities and NaN in V, some attended by a row and some behind it: every element that a row's own keys make a number is
    that number, every other is none."""
    gen = torch.Generator().manual_seed(D + Hq)
    T = sum(lens)
    q, k, v = (torch.randn(T, h, D, generator=gen).to(device=gpu_device, dtype=dtype) for h in (Hq, Hk, Hk))
    at = offsets(lens)
    for b, n in enumerate(lens):
        v[at[b] + n // 3, :, 1::4] = float("inf")       # rows from a third on
        v[at[b] + n // 2, 0, 2::8] = float("nan")       # from the middle on
        v[at[b] + n - 1, :, 3::4] = float("-inf")       # the last alone
    cu = torch.tensor(at, dtype=torch.int32, device=gpu_device)
    if page:
        kp, vp, table = _paged_of(gen, k, v, lens, page)
        o, lse = oat.omni_attention_paged(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device=gpu_device), cu,
                                          softcap=softcap, return_lse=True)
    else:
        o, lse = oat.omni_attention_packed(q, k, v, cu, softcap=softcap, return_lse=True)
    for a, e in list(zip(at, at[1:]))[:6]:
        clean = torch.where(torch.isfinite(v[a:e]), v[a:e], torch.zeros((), dtype=dtype, device=gpu_device))
        want, mean, rl = attention(q[a:e], k[a:e], clean, 0, True, softcap)
        seen = torch.cumsum((~torch.isfinite(v[a:e])).to(torch.int32), 0) > 0  # [row, Hk, D]: a key up to the row's own spoils it
        seen = seen.repeat_interleave(Hq // Hk, dim=1)
        assert torch.equal(~torch.isfinite(o[a:e]), seen)
        smax = (q[a:e].double().norm(dim=-1).max() * k[a:e].double().norm(dim=-1).max()).item() / D ** 0.5
        bound = attention_bound(want, mean, clean.double().abs().sum(0).max().item(), dtype, softcap, D, smax)
        assert bool(((o[a:e].double() - want).abs() <= bound)[~seen].all())
        assert bool(((lse[a:e].double() - rl).abs() <= (D + 8) * 2.0 ** -24 * smax + 8 * 2.0 ** -23 * softcap + 2.0 ** -21 * (1 + rl.abs())).all())


@pytest.mark.parametrize("T,Hq,Hk,D", [(4096, 8, 2, 128), (4096, 8, 8, 64), (512, 8, 8, 64), (1300, 16, 16, 128)])
@pytest.mark.parametrize("spoilt", ["first", "last"])
def test_no_numbers_do_not_stop_a_launch(gpu_device, T, Hq, Hk, D, spoilt):
    """One value that is no number, in the first key (all rows) or the last (one row): a second, slower walk over the tile's keys,
    not one for every row."""
    gen = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(T, h, D, generator=gen).to(device=gpu_device, dtype=torch.bfloat16) for h in (Hq, Hk, Hk))
    bad = v.clone()
    bad[0 if spoilt == "first" else T - 1] = float("nan")
    cu = torch.tensor([0, T], dtype=torch.int32, device=gpu_device)

    def fastest(values):
        oat.omni_attention_packed(q, k, values, cu)
        times = []
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            oat.omni_attention_packed(q, k, values, cu)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    clean, dirty = fastest(v), fastest(bad)
    # (a row at a time takes 220 - 330 times as long as the launch without; launches and clocks vary by less than 2)
    assert dirty <= 60 * clean, (clean, dirty)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Hq,Hk,D,page", [(9, 8, 8, 64, 64), (40, 8, 2, 128, 64), (64, 4, 1, 32, 16), (300, 8, 1, 64, 128), (1100, 4, 4, 32, 64)])
def test_cut_and_whole_sequences_side_by_side(gpu_device, dtype, B, Hq, Hk, D, page):
    """Single tokens whose sequences are cut into many parts, into a few and not at all, in any order, empty ones among them."""
    gen = torch.Generator().manual_seed(B)
    lens = [[1, 0, 2][0 if b % 5 else b // 5 % 3] for b in range(B)]
    kv = [(4000 + 37 * b % 1500 if b % max(B // 6, 4) == 2 else (700 if b % 7 == 1 else 60 + 11 * b % 90)) if b % 9 else 0 for b in range(B)]
    need = [-(-n // page) for n in kv]
    pool = [torch.randn(sum(need) + 1, Hk, page, D, generator=gen).to(device=gpu_device, dtype=dtype) for _ in range(2)]
    table, at = torch.zeros(B, max(need), dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n)
        at += n
    cu = offsets(lens)
    q = torch.randn(cu[-1] + 3, Hq, D, generator=gen).to(device=gpu_device, dtype=dtype)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    o, lse = oat.omni_attention_paged(q, pool[0], pool[1], table.to(gpu_device), i32(kv), i32(cu), return_lse=True)
    assert bool((o[cu[-1]:] == 0).all()) and bool((lse[cu[-1]:] == -float("inf")).all())
    at = 0
    for b, n in enumerate(need):
        rows = slice(cu[b], cu[b + 1])
        if lens[b]:
            k, v = (p[at:at + n].transpose(1, 2).reshape(-1, Hk, D)[:kv[b]] for p in pool)
            want, mean, rl = attention(q[rows], k, v, kv[b] - lens[b], True, 0.0)
            if kv[b]:
                smax = (q[rows].double().norm(dim=-1).max() * k.double().norm(dim=-1).max()).item() / D ** 0.5
                bound = attention_bound(want, mean, 0.0 if dtype == torch.bfloat16 else v.double().abs().sum(0).max().item(), dtype, 0.0, D, smax)
                assert bool(((o[rows].double() - want).abs() <= bound).all()), b
                room = (D + 8) * 2.0 ** -24 * smax + 2.0 ** -21 * (1 + rl.abs())
                live = torch.isfinite(rl)
                assert torch.equal(torch.isfinite(lse[rows]), live) and bool(((lse[rows].double() - rl).abs() <= room)[live].all()), b
            else:
                assert bool((o[rows] == 0).all()) and bool((lse[rows] == -float("inf")).all())
        at += n


def test_scratch_memory_of_many_sequences(gpu_device):
    """One call's scratch does not grow with the batch: 4096 single tokens of 32 heads."""
    B, H, D, page, dtype = 4096, 32, 128, 64, torch.bfloat16
    q = torch.zeros(B, H, D, dtype=dtype, device=gpu_device)
    kp, vp = (torch.zeros(16, H, page, D, dtype=dtype, device=gpu_device) for _ in range(2))
    table = torch.zeros(B, 16, dtype=torch.int32, device=gpu_device)
    kv = torch.full((B,), 100, dtype=torch.int32, device=gpu_device)
    cu = torch.arange(B + 1, dtype=torch.int32, device=gpu_device)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    o = oat.omni_attention_paged(q, kp, vp, table, kv, cu)
    torch.cuda.synchronize()
    assert bool((o == 0).all())
    assert torch.cuda.max_memory_allocated() - before - o.numel() * 2 <= 64 * 2 ** 20
