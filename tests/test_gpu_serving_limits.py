"""Calls of the packed-sequence operators at their limits: offsets that run backwards, values that are no numbers, scratch memory,
large groups, operands beyond 2^31 elements, an append of many sequences."""
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


@pytest.mark.parametrize("Hq,Hk,D", [(200, 1, 64), (300, 2, 32), (130, 1, 128)])
def test_more_heads_in_a_group_than_rows_in_a_tile(gpu_device, Hq, Hk, D):
    """A token's heads fill more than a tile: prompts, single tokens in parts, and gradients as the sums over single heads."""
    gen = torch.Generator().manual_seed(Hq)
    dtype, lens = torch.bfloat16, [5, 1, 90]
    T, at = sum(lens), offsets(lens)
    q, k, v, do = (torch.randn(T, h, D, generator=gen).to(device=gpu_device, dtype=dtype) for h in (Hq, Hk, Hk, Hq))
    cu = torch.tensor(at, dtype=torch.int32, device=gpu_device)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o, lse = oat.omni_attention_packed(*leaves, cu, return_lse=True)
    grads = torch.autograd.grad(o, leaves, do)
    one_by_one = [torch.zeros(t.shape, dtype=torch.float64, device=gpu_device) for t in leaves]
    size = torch.zeros(2, dtype=torch.float64)
    for h in range(0, Hq, Hq // Hk):
        for i in range(h, h + Hq // Hk, 10):
            heads, y = slice(i, min(i + 10, h + Hq // Hk)), slice(h * Hk // Hq, h * Hk // Hq + 1)
            part = [t.detach().clone().requires_grad_() for t in (q[:, heads], k[:, y], v[:, y])]
            out = oat.omni_attention_packed(*part, cu)
            # (the same products in another tile: as many keys, the same order)
            assert (out.float() - o[:, heads].float()).abs().max().item() <= 4 * 4 * torch.finfo(dtype).eps / 2
            g = torch.autograd.grad(out, part, do[:, heads])
            one_by_one[0][:, heads] = g[0].double()
            for n in (1, 2):
                one_by_one[n][:, y] += g[n].double()
                size[n - 1] += g[n].double().abs().max().item()
    # each part is rounded once, and the whole once: half a step of the largest parts
    eps = torch.finfo(dtype).eps / 2
    assert (grads[0].double() - one_by_one[0]).abs().max().item() <= 8 * eps * one_by_one[0].abs().max().item()
    for n in (1, 2):
        assert (grads[n].double() - one_by_one[n]).abs().max().item() <= 2 * eps * size[n - 1].item() + eps * grads[n].double().abs().max().item()
    kp, vp, table = _paged_of(gen, torch.randn(6000, Hk, D, generator=gen).to(device=gpu_device, dtype=dtype),
                              torch.randn(6000, Hk, D, generator=gen).to(device=gpu_device, dtype=dtype), [5000, 1000], 64)
    kv = torch.tensor([5000, 1000], dtype=torch.int32, device=gpu_device)
    cu = torch.tensor([0, 1, 3], dtype=torch.int32, device=gpu_device)
    o, lse = oat.omni_attention_paged(q[:3].detach(), kp, vp, table, kv, cu, return_lse=True)
    for b, (a, e) in enumerate(((0, 1), (1, 3))):
        n = int(kv[b])
        keys, values = (p[table[b].long()].transpose(1, 2).reshape(-1, Hk, D)[:n] for p in (kp, vp))
        want, mean, rl = attention(q[a:e].detach(), keys, values, n - (e - a), True, 0.0)
        smax = (q[a:e].double().norm(dim=-1).max() * keys.double().norm(dim=-1).max()).item() / D ** 0.5
        assert bool(((o[a:e].double() - want).abs() <= attention_bound(want, mean, 0.0, dtype, 0.0, D, smax)).all())
        assert bool(((lse[a:e].double() - rl).abs() <= (D + 8) * 2.0 ** -24 * smax + 2.0 ** -21 * (1 + rl.abs())).all())


def test_packed_rows_beyond_32_bits(gpu_device):
    """More than 2^31 elements in every operand: the last sequences, their gradients and the rows behind them."""
    gen = torch.Generator().manual_seed(3)
    dtype, H, D, n = torch.bfloat16, 64, 128, 300
    behind = 5
    T = (1 << 31) // (H * D) + 2 * n + behind
    tail = [torch.randn(2 * n, H, D, generator=gen).to(device=gpu_device, dtype=dtype) for _ in range(4)]
    lens = [700] * ((T - behind - 2 * n) // 700)
    lens += [T - behind - 2 * n - sum(lens), n, n]
    cu = torch.tensor(offsets(lens), dtype=torch.int32, device=gpu_device)
    q, k, v, do = (torch.zeros(T, H, D, dtype=dtype, device=gpu_device) for _ in range(4))
    rows = slice(T - behind - 2 * n, T - behind)
    for x, t in zip((q, k, v, do), tail):
        x[rows] = t
        x[T - behind:] = 1.0
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o, lse = oat.omni_attention_packed(*leaves, cu, return_lse=True)
    grads = torch.autograd.grad(o, leaves, do)
    assert bool((o[T - behind:] == 0).all()) and bool((lse[T - behind:] == -float("inf")).all())
    assert all(bool((g[T - behind:] == 0).all()) for g in grads)
    small = [t.clone().requires_grad_() for t in tail[:3]]
    two = torch.tensor([0, n, 2 * n], dtype=torch.int32, device=gpu_device)
    want, want_lse = oat.omni_attention_packed(*small, two, return_lse=True)
    want_grads = torch.autograd.grad(want, small, tail[3])
    # (another form may take the same rows: weights and results rounded to half a step of values of at most 6 each)
    eps = torch.finfo(dtype).eps / 2
    assert (o[rows].float() - want.float()).abs().max().item() <= 4 * 6 * eps
    assert (lse[rows] - want_lse).abs().max().item() <= 1e-4
    for g, w in zip(grads, want_grads):
        assert (g[rows].float() - w.float()).abs().max().item() <= 16 * eps * w.float().abs().max().item()
    assert bool((o[:rows.start] == 0).all())


@pytest.mark.parametrize("B", [65, 128, 129, 5000])
def test_append_of_many_sequences(gpu_device, B):
    """More sequences than a wave has lanes, some without a new token: every token finds its own."""
    gen = torch.Generator().manual_seed(B)
    dtype, Hk, D, page = torch.float16, 2, 32, 16
    lens = torch.randint(0, 4, (B,), generator=gen).tolist()
    lens[0], lens[1], lens[B - 1] = 0, 3, 2
    cached = torch.randint(0, 30, (B,), generator=gen).tolist()
    T = sum(lens) + 2
    k, v, q = (torch.randn(T, Hk, D, generator=gen).to(device=gpu_device, dtype=dtype) for _ in range(3))
    kp, vp = (torch.zeros(3 * B, Hk, page, D, dtype=dtype, device=gpu_device) for _ in range(2))
    table = torch.randperm(3 * B, generator=gen).to(torch.int32).view(B, 3)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    y = oat.omni_cache_append(k, v, kp, vp, table.to(gpu_device), i32([n + c for n, c in zip(lens, cached)]), i32(offsets(lens)), query=q)
    want_k, want_v = torch.zeros_like(kp), torch.zeros_like(vp)
    pages, at = [], []
    for b, (n, c) in enumerate(zip(lens, cached)):
        for i in range(c, c + n):
            pages.append(int(table[b, i // page]))
            at.append(i % page)
    pages, at = torch.tensor(pages, device=gpu_device), torch.tensor(at, device=gpu_device)
    want_k[pages, :, at], want_v[pages, :, at] = k[:T - 2], v[:T - 2]
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)
    assert torch.equal(y[:T - 2], q[:T - 2]) and bool((y[T - 2:] == 0).all())
