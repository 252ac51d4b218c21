"""New tokens entering a paged cache: what is written against the plain form in 64 bits, what is not written bit for bit."""
import pytest
import torch

import omni_attn_torch as oat
from serving_helpers import norm_rotate, offsets, rotate_bound

pytestmark = pytest.mark.gpu

EPS = 1e-5


def _cache(gen, device, dtype, lens, cached, Hk, D, page, spare=3):
    total = [n + c for n, c in zip(lens, cached)]
    need = [-(-n // page) for n in total]
    num = sum(need) + spare
    order = torch.randperm(num, generator=gen).to(torch.int32)
    width = max(need + [1]) + 1
    table = torch.full((len(lens), width), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    pages = [torch.randn(num, Hk, page, D, generator=gen).to(device=device, dtype=dtype) for _ in range(2)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    return table.to(device), i32(total), i32(offsets(lens)), pages


def _places(table, kv_lens, cu, page, T):
    """(page, row, position) of every token; page -1: it has no place."""
    table, kv_lens, cu = table.cpu(), kv_lens.cpu().tolist(), cu.cpu().tolist()
    out = [(-1, 0, 0)] * T
    for b in range(len(kv_lens)):
        for t in range(max(cu[b], 0), min(cu[b + 1], T)):
            pos = kv_lens[b] - cu[b + 1] + t
            if 0 <= pos < table.shape[1] * page:
                out[t] = (int(table[b, pos // page]), pos % page, pos)
    return out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,rot,Hq,Hk,page,norm,interleaved,lens,cached", [
    (128, 128, 32, 8, 64, True, False, [1] * 9, [0, 1, 63, 64, 65, 127, 200, 5, 31]),
    (64, 32, 4, 4, 16, False, True, [1, 0, 17, 100, 0, 33], [15, 3, 0, 29, 0, 1]),
    (32, 32, 6, 2, 32, True, True, [64], [0]),
    (128, 64, 8, 1, 128, True, False, [300, 1], [11, 500]),
    (96, 24, 3, 3, 16, False, False, [5, 6], [1, 2]),
    (256, 256, 2, 1, 16, True, False, [40], [3])])
def test_append(gpu_device, dtype, D, rot, Hq, Hk, page, norm, interleaved, lens, cached):
    gen = torch.Generator().manual_seed(D + len(lens))
    table, kv_lens, cu, (kp, vp) = _cache(gen, gpu_device, dtype, lens, cached, Hk, D, page)
    behind = 3  # tokens behind the last sequence
    T = sum(lens) + behind
    make = lambda H: torch.randn(T, H, D, generator=gen).to(device=gpu_device, dtype=dtype)
    q, k, v = make(Hq), make(Hk), make(Hk)
    v[0, 0, 0], v[0, 0, 1] = float("inf"), float("nan")
    w = [(1 + 0.3 * torch.randn(D, generator=gen)).to(device=gpu_device, dtype=dtype) if norm else None for _ in range(2)]
    angles = oat.omni_rotary_table(rot, max(n + c for n, c in zip(lens, cached)), device=gpu_device)
    before = kp.clone(), vp.clone()
    y = oat.omni_cache_append(k, v, kp, vp, table, kv_lens, cu, table=angles, query=q, query_norm=w[0], key_norm=w[1],
                              eps=EPS, interleaved=interleaved)
    places = _places(table, kv_lens, cu, page, T)
    position = torch.tensor([p for _, _, p in places], device=gpu_device)
    live = T - behind
    want, size = norm_rotate(q[:live], w[0], angles[position[:live]].unsqueeze(1), EPS, interleaved)
    assert bool(((y[:live].double() - want).abs() <= rotate_bound(want, size, dtype)).all())
    assert bool((y[live:] == 0).all())
    want, size = norm_rotate(k[:live], w[1], angles[position[:live]].unsqueeze(1), EPS, interleaved)
    bound = rotate_bound(want, size, dtype)
    pg = torch.tensor([p for p, _, _ in places[:live]], device=gpu_device)
    row = torch.tensor([r for _, r, _ in places[:live]], device=gpu_device)
    assert bool(((kp[pg, :, row].double() - want).abs() <= bound).all())
    bits = lambda t: t.view(torch.int16)
    assert torch.equal(bits(vp[pg, :, row]), bits(v[:live]))
    for after, old in ((kp, before[0]), (vp, before[1])):  # nothing else has changed
        after[pg, :, row] = old[pg, :, row]
        assert torch.equal(bits(after), bits(old))


def test_tokens_without_a_place_and_shared_positions(gpu_device):
    """Bad page numbers, positions before the first and behind the last page, a sequence cut short by its kv_len; rotation
    by given positions; no query; no rotation."""
    gen = torch.Generator().manual_seed(2)
    dtype, Hk, D, page = torch.bfloat16, 2, 64, 16
    lens = [3, 20, 4, 2]
    T = sum(lens)
    num = 4
    table = torch.tensor([[0, 9], [1, -1], [2, 3], [99, 99]], dtype=torch.int32, device=gpu_device)
    kv_lens = torch.tensor([2, 20, 34, 2], dtype=torch.int32, device=gpu_device)
    cu = torch.tensor(offsets(lens), dtype=torch.int32, device=gpu_device)
    k, v = (torch.randn(T, Hk, D, generator=gen).to(device=gpu_device, dtype=dtype) for _ in range(2))
    kp, vp = (torch.randn(num, Hk, page, D, generator=gen).to(device=gpu_device, dtype=dtype) for _ in range(2))
    positions = torch.randint(0, 5, (T,), generator=gen).to(gpu_device)
    angles = oat.omni_rotary_table(D, 5, device=gpu_device)
    for turned in (False, True):
        ks, vs = kp.clone(), vp.clone()
        got = oat.omni_cache_append(k, v, ks, vs, table, kv_lens, cu, table=angles if turned else None,
                                    positions=positions if turned else None)
        assert got is None
        want_k, want_v = kp.clone(), vp.clone()
        turned_k, size = norm_rotate(k, None, angles[positions].unsqueeze(1), EPS, False) if turned else (k.double(), k.double().abs())
        written = 0
        for t, (pg, row, _) in enumerate(_places(table, kv_lens, cu, page, T)):
            if 0 <= pg < num:
                written += 1
                assert bool(((ks[pg, :, row].double() - turned_k[t]).abs() <= rotate_bound(turned_k[t], size[t], dtype)).all())
                want_k[pg, :, row], want_v[pg, :, row] = ks[pg, :, row], v[t]
        assert written == 2 + 16 + 2
        assert torch.equal(ks, want_k) and torch.equal(vs, want_v)


def test_far_pages_strided_rows_and_versions(gpu_device):
    """A cache of more than 2^31 elements, its last page; rows of a fused projection; autograd learns of the change."""
    dtype, Hk, D, page = torch.float16, 8, 128, 64
    num = (1 << 31) // (Hk * D * page) + 2
    kp, vp = (torch.zeros(num, Hk, page, D, dtype=dtype, device=gpu_device) for _ in range(2))
    gen = torch.Generator().manual_seed(8)
    both = torch.randn(70, 4 * Hk, D, generator=gen).to(device=gpu_device, dtype=dtype)
    k, v = both[:, 2 * Hk:3 * Hk], both[:, 3 * Hk:]
    table = torch.tensor([[num - 1, num - 2]], dtype=torch.int32, device=gpu_device)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    version = kp._version
    oat.omni_cache_append(k, v, kp, vp, table, i32(70), i32(0, 70))
    assert kp._version > version
    for pages, x in ((kp, k), (vp, v)):
        assert torch.equal(pages[num - 1].transpose(0, 1), x[:64])
        assert torch.equal(pages[num - 2][:, :6].transpose(0, 1), x[64:])
        assert bool((pages[:num - 2] == 0).all()) and bool((pages[num - 2][:, 6:] == 0).all())
