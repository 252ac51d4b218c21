"""Gradients of the attention of packed sequences against the formula in 64 bits, and against differences."""
import math

import pytest
import torch

import omni_attn_torch as oat
from serving_helpers import half_step, offsets, smallest

pytestmark = pytest.mark.gpu


def _reference(q, k, v, do, causal, softcap, dtype):
    """One sequence: gradients in 64 bits, and how far the kernels' may be off.  Rounded are: O (through the weights of the
    forward, half a step of the mean of |v|, and itself) and so delta; P before dV; dS before dQ and dK; the results.  An
    fp16 number below the smallest normal one is off by half its smallest step.  Before that 32 bits: scores of D products,
    and products of dO and v."""
    n, Hq, D = q.shape
    Hk = k.shape[1]
    G = Hq // Hk
    h, tiny, scale = half_step(dtype) * (1 + 1e-3), smallest(dtype), 1 / math.sqrt(D)
    q, k, v, do = (t.double() for t in (q, k, v, do))
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    bounds = [torch.zeros_like(t) for t in (q, k, v)]
    smax = (q.norm(dim=-1).max() * k.norm(dim=-1).max()).item() * scale
    rel = 2 * ((D * 2.0 ** -24 + 8 * 2.0 ** -23) * smax + 16 * 2.0 ** -23 * (1 + softcap))
    for x in range(Hq):
        y = x // G
        s = (q[:, x] @ k[:, y].t()) * scale
        slope = torch.ones_like(s)
        if softcap:
            th = torch.tanh(s / softcap)
            s, slope = softcap * th, 1 - th * th
        if causal:
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), -math.inf)
        p = torch.softmax(s, -1)
        o, mean = p @ v[:, y], p @ v[:, y].abs()
        dp = do[:, x] @ v[:, y].t()
        delta = (do[:, x] * o).sum(-1, keepdim=True)
        off = (do[:, x].abs() * ((h + rel) * mean + h * o.abs() + tiny * 128 * (1 + v[:, y].abs().sum(0)))).sum(-1, keepdim=True)
        ds = p * (dp - delta) * slope
        size = do[:, x].abs() @ v[:, y].abs().t()
        # an element of dS: its own rounding, delta's, the 32-bit error of the weight and of the products
        dds = h * ds.abs() + p * slope * (off + rel * ((dp - delta).abs() + 1) + D * 2.0 ** -23 * size) + tiny
        ddp = (h + rel) * p + tiny
        grads[0][:, x] += scale * (ds @ k[:, y])
        bounds[0][:, x] += scale * (dds @ k[:, y].abs())
        grads[1][:, y] += scale * (ds.t() @ q[:, x])
        bounds[1][:, y] += scale * (dds.t() @ q[:, x].abs())
        grads[2][:, y] += p.t() @ do[:, x]
        bounds[2][:, y] += ddp.t() @ do[:, x].abs()
    return grads, [b * 1.05 + h * g.abs() + tiny + 1e-7 for b, g in zip(bounds, grads)]


def _inputs(gen, device, dtype, T, Hq, Hk, D):
    make = lambda H: torch.randn(T, H, D, generator=gen).to(device=device, dtype=dtype)
    return make(Hq), make(Hk), make(Hk), make(Hq)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("lens", [[1], [1, 0, 5, 0], [63, 64, 65, 127, 128, 129], [300, 17, 1, 41], [700], [3] * 70 + [0] * 5 + [9] * 60, [0, 0]])
@pytest.mark.parametrize("Hq,Hk,causal,softcap", [(1, 1, True, 0.0), (8, 2, True, 0.0), (6, 2, False, 0.0), (4, 4, True, 20.0),
                                                   (16, 1, False, 15.0), (3, 1, True, 0.0)])
def test_gradients(gpu_device, dtype, D, lens, Hq, Hk, causal, softcap):
    gen = torch.Generator().manual_seed(D + Hq + len(lens))
    T = sum(lens) + 2  # (two tokens behind the last sequence)
    q, k, v, do = _inputs(gen, gpu_device, dtype, T, Hq, Hk, D)
    cu = torch.tensor(offsets(lens), dtype=torch.int32, device=gpu_device)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = oat.omni_attention_packed(q, k, v, cu, causal=causal, softcap=softcap)
    with torch.no_grad():
        assert torch.equal(o, oat.omni_attention_packed(q, k, v, cu, causal=causal, softcap=softcap))
    grads = torch.autograd.grad(o, leaves, do)
    at = offsets(lens)
    for a, b in zip(at, at[1:]):
        if a == b:
            continue
        want, bound = _reference(*(t.detach()[a:b] for t in (q, k, v, do)), causal, softcap, dtype)
        for name, g, w, e in zip(("dq", "dk", "dv"), grads, want, bound):
            over = (g[a:b].double() - w).abs() - e
            assert bool((over <= 0).all()), f"{name} of the sequence at {a}: beyond its bound by {over.max().item():.3e}"
    for g in grads:
        assert bool((g[at[-1]:] == 0).all())


@pytest.mark.parametrize("softcap", [0.0, 10.0])
def test_gradients_against_differences(gpu_device, softcap):
    """The slope of sum(o u) along a direction, by central differences of the plain form in 64 bits around the very inputs."""
    from serving_helpers import attention
    gen = torch.Generator().manual_seed(3)
    dtype, lens, Hq, Hk, D = torch.float16, [50, 33], 4, 2, 64
    q, k, v, u = _inputs(gen, gpu_device, dtype, sum(lens), Hq, Hk, D)
    cu = torch.tensor(offsets(lens), dtype=torch.int32, device=gpu_device)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(oat.omni_attention_packed(q, k, v, cu, softcap=softcap), leaves, u)
    z = [torch.randn(t.shape, generator=gen).to(gpu_device).double() for t in leaves]
    at = offsets(lens)

    def loss(t):
        x = [leaf.detach().double() + t * d for leaf, d in zip(leaves, z)]
        return sum((attention(x[0][a:b], x[1][a:b], x[2][a:b], 0, True, softcap)[0] * u[a:b].double()).sum() for a, b in zip(at, at[1:]))

    step = 1e-5
    slope = ((loss(step) - loss(-step)) / (2 * step)).item()
    got = sum((g.double() * d).sum() for g, d in zip(grads, z)).item()
    room = 1e-3
    for a, b in zip(at, at[1:]):
        _, bound = _reference(*(t.detach()[a:b] for t in (q, k, v, u)), True, softcap, dtype)
        room += sum((e * d[a:b].abs()).sum() for e, d in zip(bound, z)).item()
    assert abs(slope - got) <= room, (slope, got, room)


def test_layouts_unused_inputs_and_same_bits(gpu_device):
    gen = torch.Generator().manual_seed(4)
    dtype, lens, Hq, Hk, D = torch.bfloat16, [130, 70], 8, 2, 128
    T = sum(lens)
    both = torch.randn(T, Hq + 2 * Hk, D, generator=gen).to(device=gpu_device, dtype=dtype)
    do = torch.randn(T, Hq, D, generator=gen).to(device=gpu_device, dtype=dtype)
    cu = torch.tensor(offsets(lens), dtype=torch.int32, device=gpu_device)
    flat = [t.contiguous().requires_grad_() for t in (both[:, :Hq], both[:, Hq:Hq + Hk], both[:, Hq + Hk:])]
    want = torch.autograd.grad(oat.omni_attention_packed(*flat, cu), flat, do)
    both.requires_grad_()
    o, lse = oat.omni_attention_packed(both[:, :Hq], both[:, Hq:Hq + Hk], both[:, Hq + Hk:], cu, return_lse=True)
    assert not lse.requires_grad
    got = torch.autograd.grad(o, both, do.transpose(0, 1).contiguous().transpose(0, 1))[0]
    assert torch.equal(got, torch.cat(want, 1))
    # a gradient of one input alone, an expanded one coming in
    one = torch.autograd.grad(oat.omni_attention_packed(flat[0].detach(), flat[1], flat[2].detach(), cu).float().sum(), flat[1])[0]
    ones = torch.autograd.grad(oat.omni_attention_packed(*flat, cu), flat, torch.ones_like(do))[1]
    assert torch.equal(one, ones)
    with pytest.raises(RuntimeError, match="gradients of its gradients"):
        torch.autograd.grad(oat.omni_attention_packed(*flat, cu).float().sum(), flat[0], create_graph=True)


def test_many_tiles_and_a_graph(gpu_device):
    gen = torch.Generator().manual_seed(5)
    dtype, lens, Hq, Hk, D = torch.bfloat16, [1500, 400, 33], 16, 4, 128
    T = sum(lens) + 200
    static = list(_inputs(gen, gpu_device, dtype, T, Hq, Hk, D))
    cu = torch.tensor(offsets(lens), dtype=torch.int32, device=gpu_device)

    def step():
        leaves = [t.detach().requires_grad_() for t in static[:3]]
        o = oat.omni_attention_packed(*leaves, cu)
        return [o.detach()] + list(torch.autograd.grad(o, leaves, static[3]))

    out = step()
    at = offsets(lens)
    for a, b in zip(at, at[1:]):
        want, bound = _reference(*(t[a:b] for t in static), True, 0.0, dtype)
        for g, w, e in zip(out[1:], want, bound):
            assert bool(((g[a:b].double() - w).abs() <= e).all())
    assert all(bool((g[at[-1]:] == 0).all()) for g in out)
    side = torch.cuda.Stream(device=gpu_device)
    side.wait_stream(torch.cuda.current_stream(gpu_device))
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = step()
    torch.cuda.synchronize()
    for lens in ([1500, 400, 33], [10, 900, 1000], [0, 2133, 0]):
        cu.copy_(torch.tensor(offsets(lens), dtype=torch.int32))
        for t in static:
            t.copy_(torch.randn(t.shape, generator=gen).to(dtype))
        eager = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b), lens


def test_heads_that_lie_far_apart(gpu_device):
    """Heads 2^30 elements from one another: the gradients' steps of rows reach over 3 GiB of them."""
    gen = torch.Generator().manual_seed(6)
    dtype, lens, Hq, Hk, D = torch.bfloat16, [70, 30], 2, 1, 32
    T = sum(lens)
    q, k, v, do = _inputs(gen, gpu_device, dtype, T, Hq, Hk, D)
    cu = torch.tensor(offsets(lens), dtype=torch.int32, device=gpu_device)
    far = torch.zeros((1 << 30) + T * D, dtype=dtype, device=gpu_device).as_strided((T, Hq, D), (D, 1 << 30, 1))
    near = [t.requires_grad_() for t in (q, k, v)]
    out = oat.omni_attention_packed(*near, cu)
    want = torch.autograd.grad(out, near, do)
    far.copy_(q.detach())
    leaves = [far.requires_grad_(), k, v]
    got = torch.autograd.grad(oat.omni_attention_packed(*leaves, cu), leaves, do)
    with torch.no_grad():
        assert torch.equal(oat.omni_attention_packed(far, k, v, cu), out)
        far.copy_(do)
    again = torch.autograd.grad(oat.omni_attention_packed(*near, cu), near, far.detach())
    for a, b, c in zip(want, got, again):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("B,most,Hq,Hk,D", [(70, 300, 4, 2, 64), (4500, 6, 2, 1, 32)])
def test_thousands_of_sequences(gpu_device, B, most, Hq, Hk, D):
    gen = torch.Generator().manual_seed(B)
    dtype = torch.float16
    lens = torch.randint(0, most, (B,), generator=gen).tolist()
    lens[0], lens[-1] = 0, 2
    T = sum(lens) + 40
    q, k, v, do = _inputs(gen, gpu_device, dtype, T, Hq, Hk, D)
    cu = torch.tensor(offsets(lens), dtype=torch.int32, device=gpu_device)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(oat.omni_attention_packed(*leaves, cu), leaves, do)
    at = offsets(lens)
    for a, b in list(zip(at, at[1:]))[::9] + [(at[-2], at[-1])]:
        if a == b:
            continue
        want, bound = _reference(*(t.detach()[a:b] for t in (q, k, v, do)), True, 0.0, dtype)
        for g, w, e in zip(got, want, bound):
            assert bool(((g[a:b].double() - w).abs() <= e).all()), (a, b)
    assert all(bool((g[at[-1]:] == 0).all()) and not bool(torch.isnan(g).any()) for g in got)


@pytest.mark.parametrize("causal,softcap", [(True, 0.0), (False, 0.0), (True, 15.0)])
def test_many_short_sequences_of_shared_heads(gpu_device, causal, softcap):
    """One group of waves on a tile of keys that several query heads share, at head_dim 128."""
    gen = torch.Generator().manual_seed(8)
    dtype, B, Hq, Hk, D = torch.bfloat16, 600, 8, 4, 128
    lens = [1 + 37 * b % 150 for b in range(B)]
    T = sum(lens) + 3
    q, k, v, do = _inputs(gen, gpu_device, dtype, T, Hq, Hk, D)
    cu = torch.tensor(offsets(lens), dtype=torch.int32, device=gpu_device)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(oat.omni_attention_packed(*leaves, cu, causal=causal, softcap=softcap), leaves, do)
    at = offsets(lens)
    for a, b in list(zip(at, at[1:]))[::17]:
        want, bound = _reference(*(t.detach()[a:b] for t in (q, k, v, do)), causal, softcap, dtype)
        for g, w, e in zip(got, want, bound):
            assert bool(((g[a:b].double() - w).abs() <= e).all()), (a, b)
    assert all(bool((g[at[-1]:] == 0).all()) and not bool(torch.isnan(g).any()) for g in got)
