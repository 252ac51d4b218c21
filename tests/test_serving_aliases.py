"""Keys and values of new tokens that would go to one place are refused."""
import ctypes

import pytest
import torch

import omni_attn_capi
import omni_attn_torch as oat


class Strides(ctypes.Structure):
    _fields_ = [("batch", ctypes.c_int64), ("head", ctypes.c_int64), ("row", ctypes.c_int64)]


@pytest.mark.parametrize("apart", [0, 16, 2 * 2 * 16 * 64 * 2 - 16])
def test_append_refuses_pages_that_overlap(apart):
    f = omni_attn_capi.load_library().omni_attn_cache_append_gfx950
    at, one = Strides(0, 64, 128), lambda x=0: ctypes.c_void_p(1 << 20 | x)

    def call(k_pages, v_pages):  # two pages of two heads, 16 tokens, 64 dimensions
        return f(None, one(), one(), at, at, at, None, at, k_pages, v_pages, one(), one(), one(), None, None, 0, None, None, 0, 1, 1,
                 0, 2, 64, 2, 16, 1, 0, 0, ctypes.c_float(0), 0, 1, None)

    assert call(one(), one(apart)) == 2 and call(one(apart), one()) == 2


@pytest.mark.gpu
def test_append_refuses_one_pool_for_both(gpu_device):
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn(3, 2, 64, generator=gen).to(device=gpu_device, dtype=torch.float16) for _ in range(2))
    pool = torch.zeros(2, 3, 2, 16, 64, dtype=torch.float16, device=gpu_device)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu_device)
    append = lambda kp, vp: oat.omni_cache_append(k, v, kp, vp, i32(1).view(1, 1), i32(3), i32(0, 3))
    for kp, vp in ((pool[0], pool[0]), (pool.view(6, 2, 16, 64)[:3], pool.view(6, 2, 16, 64)[2:5])):
        with pytest.raises(ValueError, match="overlap"):
            append(kp, vp)
    assert bool((pool == 0).all())
    append(pool[0], pool[1])  # halves of one tensor are apart
    assert torch.equal(pool[0, 1, :, :3].transpose(0, 1), k) and torch.equal(pool[1, 1, :, :3].transpose(0, 1), v)
