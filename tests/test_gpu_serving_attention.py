"""Attention of packed sequences, over their own keys and over a paged cache, against the plain form in 64 bits: every
kernel (few rows and tiles, whole and in parts), head layouts, lengths from nothing to long ones, stale and bad pages."""
import math

import pytest
import torch

import omni_attn_torch as oat
from serving_helpers import attention, attention_bound, offsets

pytestmark = pytest.mark.gpu


def _compare(o, lse, q, seqs, causal, softcap, dtype, what):
    """seqs: (first token, tokens, k, v) per sequence, k and v [kv, Hk, D]."""
    D = q.shape[-1]
    assert o.shape == q.shape and o.dtype == dtype and lse.dtype == torch.float32 and lse.shape == q.shape[:2]
    covered = 0
    for t0, n, k, v in seqs:
        covered = max(covered, t0 + n)
        if n == 0:
            continue
        ro, mean, rl = attention(q[t0:t0 + n], k, v, k.shape[0] - n, causal, softcap)
        go, gl = o[t0:t0 + n].double(), lse[t0:t0 + n].double()
        empty = torch.isinf(rl)
        assert torch.equal(torch.isinf(gl) & (gl < 0), empty), f"{what}: rows without a key differ"
        assert bool((go[empty] == 0).all()), what
        if k.shape[0] == 0:
            continue
        smax = (q[t0:t0 + n].double().norm(dim=-1).max() * k.double().norm(dim=-1).max()).item() / math.sqrt(D)
        vmax = v.double().abs().sum(0).max().item()
        over = (go - ro).abs() - attention_bound(ro, mean, vmax, dtype, softcap, D, smax)
        assert bool((over <= 0).all()), f"{what}: sequence at {t0} beyond its bound by {over.max().item():.3e}"
        # a logsumexp is a score and a logarithm in 32 bits
        room = (D + 8) * 2.0 ** -24 * smax + 8 * 2.0 ** -23 * softcap + 2.0 ** -21 * (1 + rl[~empty].abs())
        assert bool(((gl - rl)[~empty].abs() <= room).all()), f"{what}: logsumexp"
    assert bool((o[covered:] == 0).all()) and bool(torch.isinf(lse[covered:]).all()), f"{what}: rows behind the last sequence"


def _packed(gen, device, dtype, lens, Hq, Hk, D, behind=2):
    T = sum(lens) + behind
    make = lambda H: torch.randn(T, H, D, generator=gen).to(device=device, dtype=dtype)
    return make(Hq), make(Hk), make(Hk), torch.tensor(offsets(lens), dtype=torch.int32, device=device)


LENS = {
    "one": [1], "empty_between": [1, 0, 5, 0], "tile_borders": [63, 64, 65, 127, 128, 129], "prompts": [300, 17, 1, 41],
    "long": [1000], "short_many": [3] * 70 + [0] * 5 + [9] * 60, "none": [0, 0],
}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("Hq,Hk,causal,softcap", [(1, 1, True, 0.0), (8, 2, True, 0.0), (6, 2, False, 0.0), (8, 8, True, 20.0),
                                                   (16, 1, False, 15.0), (3, 1, True, 0.0)])
def test_packed(gpu_device, dtype, D, lens, Hq, Hk, causal, softcap):
    gen = torch.Generator().manual_seed(D + Hq)
    n = LENS[lens]
    q, k, v, cu = _packed(gen, gpu_device, dtype, n, Hq, Hk, D)
    o, lse = oat.omni_attention_packed(q, k, v, cu, causal=causal, softcap=softcap, return_lse=True)
    at = offsets(n)
    _compare(o, lse, q, [(a, b - a, k[a:b], v[a:b]) for a, b in zip(at, at[1:])], causal, softcap, dtype, lens)
    assert torch.equal(oat.omni_attention_packed(q, k, v, cu, causal=causal, softcap=softcap), o)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,Hq,Hk,D", [
    ([1500, 2048, 700, 33, 128, 1], 32, 8, 128),   # tiles, whole: their order goes by length
    ([1024] * 3, 16, 16, 64), ([2000, 100], 24, 24, 32),
    ([40] * 330, 8, 8, 64),                        # few rows, whole
    ([1300], 16, 16, 128), ([700, 0, 900, 64], 32, 8, 64), ([1500], 12, 12, 32)])  # two groups of waves on tiles of 64 rows
@pytest.mark.parametrize("causal,softcap", [(True, 0.0), (False, 20.0)])
def test_packed_whole_tiles(gpu_device, dtype, lens, Hq, Hk, D, causal, softcap):
    gen = torch.Generator().manual_seed(Hq)
    q, k, v, cu = _packed(gen, gpu_device, dtype, lens, Hq, Hk, D, behind=300)
    o, lse = oat.omni_attention_packed(q, k, v, cu, causal=causal, softcap=softcap, return_lse=True)
    at = offsets(lens)
    _compare(o, lse, q, [(a, b - a, k[a:b], v[a:b]) for a, b in zip(at, at[1:])], causal, softcap, dtype, "whole")


def test_packed_rows_of_a_fused_projection(gpu_device):
    gen = torch.Generator().manual_seed(1)
    dtype, T, Hq, Hk, D = torch.bfloat16, 200, 8, 2, 64
    both = torch.randn(T, Hq + 2 * Hk, D, generator=gen).to(device=gpu_device, dtype=dtype)
    q, k, v = both[:, :Hq], both[:, Hq:Hq + Hk], both[:, Hq + Hk:]
    cu = torch.tensor([0, 120, 200], dtype=torch.int32, device=gpu_device)
    want = oat.omni_attention_packed(q.contiguous(), k.contiguous(), v.contiguous(), cu, return_lse=True)
    for x in ((q, k, v), (q, k.contiguous(), v), (torch.cat([q, q], -1)[..., :D], k, v.transpose(0, 1).contiguous().transpose(0, 1))):
        got = oat.omni_attention_packed(*x, cu, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.empty(T, Hq, D + 1, dtype=dtype, device=gpu_device)[..., 1:]  # copied
    odd.copy_(q)
    assert torch.equal(oat.omni_attention_packed(odd, k, v, cu), want[0])


def test_packed_agrees_with_the_block_sparse_operator(gpu_device):
    """One sequence per batch element, as many key heads as query heads, a causal block mask: the same function."""
    gen = torch.Generator().manual_seed(12)
    dtype, B, H, S, D = torch.bfloat16, 2, 4, 512, 128
    q, k, v = (torch.randn(B, S, H, D, generator=gen).to(device=gpu_device, dtype=dtype) for _ in range(3))
    mask = oat.create_causal_omni_block_mask(B, H, S, S, device=gpu_device)
    ref = oat.omni_attention(*(t.transpose(1, 2) for t in (q, k, v)), mask).transpose(1, 2)
    cu = torch.arange(0, B * S + 1, S, dtype=torch.int32, device=gpu_device)
    got = oat.omni_attention_packed(*(t.reshape(B * S, H, D) for t in (q, k, v)), cu).view(B, S, H, D)
    # two roundings of weights and results, each half a step of values of at most 4
    assert (got.float() - ref.float()).abs().max().item() <= 4 * 4 * torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,Hq,Hk,D", [([200], 4, 2, 64), ([1300], 16, 16, 128), ([1500, 2048, 700], 32, 8, 128), ([9] * 40, 8, 8, 32)])
def test_scores_that_outgrow_their_reference(gpu_device, dtype, lens, Hq, Hk, D):
    """Scores that grow along the keys, in steps and within a step, shrink, and jump at a single key."""
    gen = torch.Generator().manual_seed(13)
    q, k, v, cu = _packed(gen, gpu_device, dtype, lens, Hq, Hk, D)
    position = torch.cat([torch.arange(n) for n in lens] + [torch.zeros(2, dtype=torch.long)]).to(gpu_device)
    towards = torch.randn(D, generator=gen).to(gpu_device)
    size = 0.02 * position.float() * torch.where(position % 97 == 50, 6.0, 1.0) * torch.where(position > 1000, 0.3, 1.0)
    k = (k.float() + size.clamp(max=25.0).view(-1, 1, 1) * towards / towards.norm()).to(dtype)
    q = (q.float() + 4 * towards / towards.norm()).to(dtype)
    at = offsets(lens)
    for softcap in (0.0, 30.0):
        o, lse = oat.omni_attention_packed(q, k, v, cu, softcap=softcap, return_lse=True)
        _compare(o, lse, q, [(a, b - a, k[a:b], v[a:b]) for a, b in zip(at, at[1:])], True, softcap, dtype, "growing")


def _paged(gen, device, dtype, lens, kv, Hq, Hk, D, page, behind=2, spare=2):
    T = sum(lens) + behind
    q = torch.randn(T, Hq, D, generator=gen).to(device=device, dtype=dtype)
    need = [-(-n // page) for n in kv]
    num = sum(need) + spare
    order = torch.randperm(num, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(need + [1]) + 2), 2 ** 30, dtype=torch.int32)  # (bad numbers behind each sequence)
    pools = [torch.full((num, Hk, page, D), float("nan"), dtype=dtype, device=device) for _ in range(2)]
    keys, at = [], 0
    for b, n in enumerate(kv):
        table[b, :need[b]] = order[at:at + need[b]]
        own = order[at:at + need[b]].long().to(device)
        at += need[b]
        rows = [torch.randn(n, Hk, D, generator=gen).to(device=device, dtype=dtype) for _ in range(2)]
        for pool, x in zip(pools, rows):  # (rows behind the sequence stay NaN)
            wide = torch.full((need[b] * page, Hk, D), float("nan"), dtype=dtype, device=device)
            wide[:n] = x
            if need[b]:
                pool[own] = wide.view(need[b], page, Hk, D).transpose(1, 2)
        keys.append(rows)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    return q, pools, table.to(device), i32(kv), i32(offsets(lens)), keys


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("lens,kv,Hq,Hk,causal,softcap", [
    ([1], [1], 8, 8, True, 0.0), ([1], [700], 32, 8, True, 0.0),
    ([1] * 7, [1, 15, 16, 17, 500, 64, 1111], 8, 2, True, 0.0), ([1, 0, 1, 1], [90, 33, 0, 5], 4, 1, True, 20.0),
    ([3, 1, 8], [3, 130, 77], 6, 2, True, 0.0), ([5, 2], [5, 300], 4, 4, False, 0.0),
    ([70, 200, 1], [1500, 200, 40], 8, 2, True, 0.0), ([130], [900], 2, 1, False, 30.0),
    ([600, 500], [900, 700], 16, 8, True, 0.0), ([600, 1, 500], [600, 0, 1000], 8, 8, False, 20.0),
    ([4, 40], [2, 30], 2, 2, True, 0.0)])  # (fewer keys than tokens: the first tokens have none)
def test_paged(gpu_device, dtype, D, page, lens, kv, Hq, Hk, causal, softcap):
    gen = torch.Generator().manual_seed(page + D + len(lens))
    q, (kp, vp), table, kv_lens, cu, keys = _paged(gen, gpu_device, dtype, lens, kv, Hq, Hk, D, page)
    o, lse = oat.omni_attention_paged(q, kp, vp, table, kv_lens, cu, causal=causal, softcap=softcap, return_lse=True)
    at = offsets(lens)
    _compare(o, lse, q, [(at[b], lens[b], *keys[b]) for b in range(len(lens))], causal, softcap, dtype, f"page {page}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_paged_many_sequences_and_long_ones(gpu_device, dtype):
    gen = torch.Generator().manual_seed(4)
    for lens, kv, Hq, Hk, D in (([1] * 150, [1 + 37 * i % 400 for i in range(150)], 8, 2, 64), ([1, 1], [30000, 3], 16, 2, 128),
                                ([260, 1], [9000, 20], 4, 1, 128)):
        q, (kp, vp), table, kv_lens, cu, keys = _paged(gen, gpu_device, dtype, lens, kv, Hq, Hk, D, 32)
        o, lse = oat.omni_attention_paged(q, kp, vp, table, kv_lens, cu, return_lse=True)
        at = offsets(lens)
        _compare(o, lse, q, [(at[b], lens[b], *keys[b]) for b in range(len(lens))], True, 0.0, dtype, str(kv[:3]))


@pytest.mark.parametrize("lens,kv,Hq,Hk,D", [([1, 6, 3], [50, 6, 90], 4, 2, 64), ([200, 90], [200, 300], 4, 2, 64),
                                             ([600, 500], [900, 700], 16, 8, 128), ([7] * 200, [60] * 200, 8, 8, 32),
                                             ([400], [6000], 4, 1, 128), ([9, 2], [5000, 700], 8, 2, 128)])
def test_values_that_are_no_numbers_behind_a_row(gpu_device, lens, kv, Hq, Hk, D):
    """Infinities and NaN in K and V of later keys of the same sequence reach no row that does not attend them."""
    gen = torch.Generator().manual_seed(7)
    dtype, page = torch.bfloat16, 16
    q, (kp, vp), table, kv_lens, cu, keys = _paged(gen, gpu_device, dtype, lens, kv, Hq, Hk, D, page)
    clean = oat.omni_attention_paged(q, kp, vp, table, kv_lens, cu)
    at = offsets(lens)
    for b, n in enumerate(lens):
        if n < 2:
            continue
        last = kv[b] - 1 - n // 4  # this key and what is behind it is spoilt
        pos = torch.arange(last, kv[b], device=gpu_device)
        pg = table[b][pos // page].long()
        bad = torch.where(pos % 2 == 1, float("inf"), float("nan")).to(dtype)
        vp[pg, :, pos % page, ::3] = bad.view(-1, 1, 1).expand(-1, Hk, len(range(0, D, 3)))
        third = pos[pos % 3 == 0]
        kp[table[b][third // page].long(), :, third % page] = float("nan")
    dirty = oat.omni_attention_paged(q, kp, vp, table, kv_lens, cu)
    for b, n in enumerate(lens):
        first_bad = n - 1 - n // 4 if n >= 2 else n
        a = at[b]
        # (a row may be summed in another order once a neighbour is spoilt)
        diff = (clean[a:a + first_bad].float() - dirty[a:a + first_bad].float()).abs()
        assert bool((diff <= 4 * torch.finfo(dtype).eps).all()), b
        if n >= 2:
            assert not bool(torch.isfinite(dirty[a + first_bad:a + n, :, 0]).any())  # (an infinity alone stays one)


def test_bad_pages_do_not_fault_and_far_pages_are_read(gpu_device):
    dtype, Hk, D, page = torch.float16, 8, 128, 64
    num = (1 << 31) // (Hk * D * page) + 2  # more than 2^31 elements
    kp, vp = (torch.zeros(num, Hk, page, D, dtype=dtype, device=gpu_device) for _ in range(2))
    gen = torch.Generator().manual_seed(3)
    for pool in (kp, vp):
        pool[num - 2:] = torch.randn(2, Hk, page, D, generator=gen).to(device=gpu_device, dtype=dtype)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    q = torch.randn(101, 16, D, generator=gen).to(device=gpu_device, dtype=dtype)
    keys = [pool[num - 2:].transpose(1, 2).reshape(2 * page, Hk, D) for pool in (kp, vp)]
    for table in ([[num - 2, num - 1, -1]] * 2, [[num - 2, 2 ** 31 - 1, 5]] * 2):  # (a number beyond the cache is its last page)
        for lens in ([1, 1], [100, 1]):
            T = sum(lens)
            o, lse = oat.omni_attention_paged(q[:T], kp, vp, i32(table), i32([100, 128]), i32(offsets(lens)), return_lse=True)
            at = offsets(lens)
            seqs = [(at[b], lens[b], keys[0][:n], keys[1][:n]) for b, n in enumerate((100, 128))]
            _compare(o, lse, q[:T], seqs, True, 0.0, dtype, "far")
    # lengths beyond the page table and below zero are cut, offsets that run backwards are empty sequences
    o = oat.omni_attention_paged(q[:2], kp, vp, i32([[num - 2], [0]]), i32([10 ** 6, -5]), i32([0, 1, 2]))
    want = oat.omni_attention_paged(q[:1], kp, vp, i32([[num - 2]]), i32([64]), i32([0, 1]))
    assert torch.equal(o[:1], want) and bool((o[1] == 0).all())
    oat.omni_attention_paged(q[:9], kp, vp, i32([[0], [1]]), i32([64, 64]), i32([7, 2, 500]))
    torch.cuda.synchronize()


def test_graph_replay_with_other_lengths_and_another_stream(gpu_device):
    """Lengths and pages are read on the device: a captured step serves other lengths, and two captured steps that use
    one after the other do not disturb each other."""
    gen = torch.Generator().manual_seed(10)
    dtype, B, Hq, Hk, D, page = torch.bfloat16, 5, 8, 2, 64, 16
    kp, vp = (torch.randn(B * 40, Hk, page, D, generator=gen).to(device=gpu_device, dtype=dtype) for _ in range(2))
    table = torch.randperm(B * 40, generator=gen).to(torch.int32).view(B, 40).to(gpu_device)
    cu = torch.arange(B + 1, dtype=torch.int32, device=gpu_device)
    q = torch.randn(B, Hq, D, generator=gen).to(device=gpu_device, dtype=dtype)
    k, v = (torch.randn(B, Hk, D, generator=gen).to(device=gpu_device, dtype=dtype) for _ in range(2))
    kv_lens = torch.full((B,), 17, dtype=torch.int32, device=gpu_device)
    angles = oat.omni_rotary_table(D, 640, device=gpu_device)

    def step():
        y = oat.omni_cache_append(k, v, kp, vp, table, kv_lens, cu, table=angles, query=q)
        return oat.omni_attention_paged(y, kp, vp, table, kv_lens, cu, return_lse=True)

    side = torch.cuda.Stream(device=gpu_device)
    side.wait_stream(torch.cuda.current_stream(gpu_device))
    with torch.cuda.stream(side):
        on_side = step()
    side.synchronize()
    for a, b in zip(on_side, step()):
        assert torch.equal(a, b)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph, stream=side):
            outs.append(step())
    torch.cuda.synchronize()
    for rep in range(4):
        kv_lens.copy_(torch.randint(1, 640, (B,), generator=gen).to(torch.int32))
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen).to(dtype))
        eager = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            for a, b in zip(out, eager):
                assert torch.equal(a, b), rep


def test_two_streams_at_once(gpu_device):
    """Calls that run at the same time have workspaces of their own."""
    gen = torch.Generator().manual_seed(14)
    dtype, lens, kv, Hq, Hk, D = torch.bfloat16, [1, 1, 3], [9000, 700, 4000], 8, 2, 128
    made = [_paged(gen, gpu_device, dtype, lens, kv, Hq, Hk, D, 32) for _ in range(2)]
    call = lambda m: oat.omni_attention_paged(m[0], m[1][0], m[1][1], m[2], m[3], m[4], return_lse=True)
    want = [call(m) for m in made]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=gpu_device) for _ in made]
    for rep in range(5):
        got = []
        for stream, m in zip(streams, made):
            with torch.cuda.stream(stream):
                got.append([call(m) for _ in range(4)])
        torch.cuda.synchronize()
        for w, calls in zip(want, got):
            for c in calls:
                assert torch.equal(c[0], w[0]) and torch.equal(c[1], w[1]), rep


def test_refusals_on_the_gpu(gpu_device):
    gen = torch.Generator().manual_seed(15)
    q, (kp, vp), table, kv_lens, cu, _ = _paged(gen, gpu_device, torch.float16, [1, 2], [20, 30], 4, 2, 64, 16)
    paged = lambda **x: oat.omni_attention_paged(*[x.get(n, d) for n, d in (("q", q), ("kp", kp), ("vp", vp), ("table", table), ("kv", kv_lens), ("cu", cu))],
                                                 softcap=x.get("softcap", 0.0))
    rows = q[:, :2].contiguous()
    append = lambda **x: oat.omni_cache_append(x.get("k", rows), rows, x.get("kp", kp), vp, table, kv_lens, cu, **x.get("more", {}))
    packed = lambda **x: oat.omni_attention_packed(x.get("q", q), x.get("k", rows), x.get("v", rows), x.get("cu", cu))
    angles = oat.omni_rotary_table(64, 40, device=gpu_device)
    for call, match in (
            (lambda: paged(q=q.float()), "float16"), (lambda: paged(q=q.bfloat16()), "dtype"), (lambda: paged(q=q[:, :3]), "multiple"),
            (lambda: paged(q=q[:, :, :48]), "head_dim"), (lambda: paged(kp=kp[:, :, :12].contiguous(), vp=vp[:, :, :12].contiguous()), "page_size"),
            (lambda: paged(kp=kp[:, :, :8].contiguous(), vp=vp[:, :, :8].contiguous()), "page_size"),
            (lambda: paged(kp=kp.transpose(1, 2), vp=vp.transpose(1, 2)), "contiguous"), (lambda: paged(table=table.long()), "int32"),
            (lambda: paged(kv=kv_lens[:1]), "cu_seqlens"), (lambda: paged(cu=cu.cpu()), "device"), (lambda: paged(table=table[:1]), "row per"),
            (lambda: paged(softcap=-1.0), "softcap"), (lambda: paged(softcap=float("nan")), "softcap"), (lambda: paged(q=q.cpu()), "GPU"),
            (lambda: paged(q=q.detach().requires_grad_()), "no_grad"), (lambda: append(k=rows.detach().requires_grad_()), "no_grad"),
            (lambda: append(more=dict(query_norm=torch.ones(64, dtype=torch.float16, device=gpu_device))), "query"),
            (lambda: append(more=dict(positions=cu[:1])), "table"), (lambda: append(more=dict(table=angles[:, :12])), "rotary_dim"),
            (lambda: append(more=dict(table=angles.double())), "float32"), (lambda: append(more=dict(table=angles, positions=cu)), "one entry"),
            (lambda: append(k=rows[:, :1]), "kv_heads"), (lambda: packed(k=rows[:1]), "kv_heads"), (lambda: packed(cu=cu[:0]), "entry"),
            (lambda: packed(v=rows.bfloat16()), "dtype"),
            (lambda: oat.omni_qk_rotary(q, rows, cu, angles), "one entry"), (lambda: oat.omni_qk_rotary(q, rows[:1], cu, angles), "tokens"),
            (lambda: oat.omni_qk_rotary(q[..., :60], rows[..., :60], torch.zeros(5, dtype=torch.int64, device=gpu_device), angles), "head_dim"),
            (lambda: oat.omni_qk_rotary(q, rows, torch.zeros(5, device=gpu_device), angles), "int32"),
            (lambda: oat.omni_qk_rotary(q, rows, torch.zeros(5, dtype=torch.int64, device=gpu_device), angles, eps=-1.0), "eps"),
            (lambda: oat.omni_qk_rotary(q, rows, torch.zeros(5, dtype=torch.int64, device=gpu_device), angles,
                                        key_norm=torch.ones(32, dtype=torch.float16, device=gpu_device)), "key_norm")):
        with pytest.raises(ValueError, match=match):
            call()
    with torch.inference_mode():  # pages made here may be written here
        inside = kp.clone(), vp.clone()
        oat.omni_cache_append(rows, rows, *inside, table, kv_lens, cu)
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        oat.omni_cache_append(rows, rows, *inside, table, kv_lens, cu)
    with torch.no_grad():
        paged(q=q.detach().requires_grad_())


@pytest.mark.parametrize("B,kv,page,Hq,Hk,D", [(65, 1500, 64, 4, 1, 128), (513, 900, 64, 4, 1, 128), (1100, 700, 128, 8, 2, 64), (4500, 520, 16, 2, 1, 32)])
def test_paged_thousands_of_sequences(gpu_device, B, kv, page, Hq, Hk, D):
    """More sequences than the waves count by themselves: parts, tokens that a sequence has none or several of."""
    gen = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 4, (B,), generator=gen).tolist()
    keys = torch.randint(0, kv, (B,), generator=gen).tolist()
    keys[B // 2] = 8 * kv  # one that is cut into many parts
    lens[B // 2], lens[-1] = 20, 1
    dtype = torch.bfloat16
    q, (kp, vp), table, kv_lens, cu, rows = _paged(gen, gpu_device, dtype, lens, keys, Hq, Hk, D, page, behind=70)
    o, lse = oat.omni_attention_paged(q, kp, vp, table, kv_lens, cu, return_lse=True)
    at = offsets(lens)
    looked_at = [b for b in range(B) if b % 5 == 0 or b in (B // 2, B - 1)]
    _compare(o, lse, q, [(at[b], lens[b], *rows[b]) for b in looked_at], True, 0.0, dtype, str(B))
    assert not bool(torch.isnan(o).any()) and not bool(torch.isnan(lse).any())  # (no row is left out)
    assert torch.equal(oat.omni_attention_paged(q, kp, vp, table, kv_lens, cu), o)


@pytest.mark.parametrize("B,most,Hq,Hk,D", [(70, 300, 8, 2, 64), (513, 40, 4, 4, 128), (4500, 9, 6, 2, 32)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_thousands_of_sequences(gpu_device, B, most, Hq, Hk, D, causal):
    gen = torch.Generator().manual_seed(B)
    lens = torch.randint(0, most, (B,), generator=gen).tolist()
    lens[0], lens[-1] = 0, 2
    dtype = torch.float16
    q, k, v, cu = _packed(gen, gpu_device, dtype, lens, Hq, Hk, D, behind=100)
    o, lse = oat.omni_attention_packed(q, k, v, cu, causal=causal, return_lse=True)
    at = offsets(lens)
    spans = list(zip(at, at[1:]))
    _compare(o, lse, q, [(a, b - a, k[a:b], v[a:b]) for a, b in spans[::7] + spans[-1:]], causal, 0.0, dtype, str(B))
    assert not bool(torch.isnan(o).any()) and not bool(torch.isnan(lse).any())
    assert torch.equal(oat.omni_attention_packed(q, k, v, cu, causal=causal), o)


def test_paged_chunks_of_many_sequences(gpu_device):
    """Tiles of 128 rows in parts, more sequences than a wave has lanes."""
    gen = torch.Generator().manual_seed(9)
    B, Hq, Hk, D, dtype = 70, 4, 1, 64, torch.float16
    lens = [40 + 3 * b % 50 for b in range(B)]
    keys = [n + 100 + 211 * b % 3500 for b, n in enumerate(lens)]
    q, (kp, vp), table, kv_lens, cu, rows = _paged(gen, gpu_device, dtype, lens, keys, Hq, Hk, D, 64)
    at = offsets(lens)
    for causal in (True, False):
        o, lse = oat.omni_attention_paged(q, kp, vp, table, kv_lens, cu, causal=causal, return_lse=True)
        _compare(o, lse, q, [(at[b], lens[b], *rows[b]) for b in range(0, B, 3)] + [(at[-2], lens[-1], *rows[-1])], causal, 0.0, dtype, "chunks")
        assert not bool(torch.isnan(o).any()) and not bool(torch.isnan(lse).any())


@pytest.mark.parametrize("B,Hq,Hk,D,softcap", [(30, 4, 1, 128, 0.0), (85, 4, 1, 128, 0.0), (40, 8, 2, 64, 20.0), (64, 5, 1, 32, 0.0)])
def test_parts_of_uneven_sequences(gpu_device, B, Hq, Hk, D, softcap):
    """Tiles of 128 rows, one sequence cut into many parts and the others into few or none; heads of a token in two tiles;
    sequences without tokens and without keys among them."""
    gen = torch.Generator().manual_seed(B + D)
    dtype = torch.bfloat16
    lens = [0 if b % 7 == 3 else 60 + 5 * b % 70 for b in range(B)]
    keys = [0 if b % 11 == 5 else lens[b] + 37 * b % 230 for b in range(B)]
    keys[B // 2] = 3500
    q, (kp, vp), table, kv_lens, cu, rows = _paged(gen, gpu_device, dtype, lens, keys, Hq, Hk, D, 64, behind=130)
    at = offsets(lens)
    for causal in (True, False):
        o, lse = oat.omni_attention_paged(q, kp, vp, table, kv_lens, cu, causal=causal, softcap=softcap, return_lse=True)
        _compare(o, lse, q, [(at[b], lens[b], *rows[b]) for b in range(B)], causal, softcap, dtype, "parts")
        assert torch.equal(oat.omni_attention_paged(q, kp, vp, table, kv_lens, cu, causal=causal, softcap=softcap), o)


@pytest.mark.parametrize("lens,cached,Hq,Hk,D", [([100], [20000], 8, 1, 128), ([512, 300], [3000, 1401], 8, 2, 64),
                                                 ([40, 300, 7, 0, 200], [6000, 0, 2500, 900, 64], 3, 1, 32), ([33] * 16, [1000 + 700 * b for b in range(16)], 8, 1, 64)])
@pytest.mark.parametrize("page", [32, 64])
def test_chunks_in_weighed_parts(gpu_device, lens, cached, Hq, Hk, D, page):
    gen = torch.Generator().manual_seed(D + page)
    dtype = torch.float16
    keys = [n + m for n, m in zip(lens, cached)]
    q, (kp, vp), table, kv_lens, cu, rows = _paged(gen, gpu_device, dtype, lens, keys, Hq, Hk, D, page, behind=3)
    at = offsets(lens)
    for causal in (True, False):
        o, lse = oat.omni_attention_paged(q, kp, vp, table, kv_lens, cu, causal=causal, return_lse=True)
        _compare(o, lse, q, [(at[b], lens[b], *rows[b]) for b in range(len(lens))], causal, 0.0, dtype, "weighed")
