"""Calls of the packed-sequence operators at their limits: offsets that run backwards."""
import pytest
import torch

import omni_attn_torch as oat

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
