"""Norm and rotation of query and key heads against the plain form in 64 bits: both pair layouts, part of the head, norms,
layouts in memory, positions, gradients against the formula's and against differences."""
import pytest
import torch

import omni_attn_torch as oat
from serving_helpers import half_step, norm_rotate, rotate_bound, smallest

pytestmark = pytest.mark.gpu

EPS = 1e-5


def _inputs(gen, device, dtype, shape_q, shape_k, D, norm, weight_dtype=None):
    q = torch.randn(shape_q, generator=gen).to(device=device, dtype=dtype)
    k = (3 * torch.randn(shape_k, generator=gen)).to(device=device, dtype=dtype)
    w = [(1 + 0.3 * torch.randn(D, generator=gen)).to(device=device, dtype=weight_dtype or dtype) if norm else None for _ in range(2)]
    return q, k, w[0], w[1]


def _check(got, x, w, angles, interleaved, dtype, what):
    want, magnitude = norm_rotate(x, w, angles, EPS, interleaved)
    over = (got.double() - want).abs() - rotate_bound(want, magnitude, dtype)
    assert bool((over <= 0).all()), f"{what}: beyond its bound by {over.max().item():.3e}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot,norm,Hq,Hk,S", [
    (128, 128, True, 32, 8, 77), (128, 64, False, 5, 1, 3), (64, 64, False, 8, 8, 512), (64, 32, True, 3, 2, 130),
    (32, 32, True, 4, 4, 65), (32, 8, False, 1, 1, 1), (96, 96, True, 7, 7, 33), (96, 24, True, 2, 1, 9),
    (256, 128, True, 2, 2, 20), (256, 256, False, 40, 3, 5), (8, 8, True, 6, 6, 17), (80, 40, True, 70, 70, 4),
    (248, 8, True, 3, 1, 6)])
def test_rotary_forward_and_backward(gpu_device, dtype, interleaved, D, rot, norm, Hq, Hk, S):
    gen = torch.Generator().manual_seed(D * 1000 + S)
    B = 2
    q, k, wq, wk = _inputs(gen, gpu_device, dtype, (B, Hq, S, D), (B, Hk, S, D), D, norm)
    table = oat.omni_rotary_table(rot, S + 5, device=gpu_device)
    positions = torch.randint(0, S + 5, (B, S), generator=gen).to(gpu_device)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk) if t is not None]
    yq, yk = oat.omni_qk_rotary(q, k, positions, table, wq, wk, EPS, interleaved)
    angles = table[positions].unsqueeze(1)
    for got, x, w, name in ((yq, q, wq, "query"), (yk, k, wk, "key")):
        assert got.shape == x.shape and got.dtype == dtype
        _check(got.detach(), x.detach(), None if w is None else w.detach(), angles, interleaved, dtype, name)
    dyq = torch.randn(q.shape, generator=gen).to(device=gpu_device, dtype=dtype)
    dyk = torch.randn(k.shape, generator=gen).to(device=gpu_device, dtype=dtype)
    grads = torch.autograd.grad([yq, yk], leaves, [dyq, dyk])
    wide = [t.detach().double().requires_grad_() for t in leaves]
    outs = [norm_rotate(wide[0], wide[2] if norm else None, angles, EPS, interleaved)[0],
            norm_rotate(wide[1], wide[3] if norm else None, angles, EPS, interleaved)[0]]
    want = torch.autograd.grad(outs, wide, [dyq.double(), dyk.double()])
    for i, (got, ref) in enumerate(zip(grads, want)):
        assert got.shape == ref.shape and got.dtype == leaves[i].dtype
        if i < 2:
            # dx = r (g w - n (g w . n) / D): terms of at most r |g| |w| and, since |n|^2 = D, as much again on average
            x, w, dy = wide[i].detach(), (wide[2 + i].detach() if norm else None), (dyq, dyk)[i].double()
            r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) if norm else torch.ones_like(x[..., :1])
            gw = dy.abs().amax(-1, keepdim=True) * 2 * (w.abs().max() if norm else 1.0)
            size = r * gw * (1 + (x * r).abs() if norm else 1.0)
            bound = half_step(dtype) * ref.abs() * (1 + 1e-3) + 60 * 2.0 ** -24 * size + smallest(dtype)
        else:
            # sums over B * S * H rows in 32 bits: each term once rounded, and the sums of a lane's rows
            x, dy = wide[i - 2].detach(), (dyq, dyk)[i - 2].double()
            n = (x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)).abs()
            terms = (n * 2 * dy.abs().amax(-1, keepdim=True)).sum((0, 1, 2))
            rows = B * S * x.shape[1]
            bound = half_step(dtype) * ref.abs() * (1 + 1e-3) + (40 + min(rows, 64)) * 2.0 ** -24 * terms + smallest(dtype)
        over = (got.double() - ref).abs() - bound
        assert bool((over <= 0).all()), f"gradient {i}: beyond its bound by {over.max().item():.3e}"


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_against_differences(gpu_device, interleaved):
    """The directional derivative of sum(y u) along (x, w) -> (x + t z, w + t s), by central differences of the plain form
    in 64 bits around the very inputs, against the kernels' gradients."""
    gen = torch.Generator().manual_seed(5)
    dtype, B, H, S, D, rot = torch.float16, 1, 3, 21, 64, 32
    q, k, wq, wk = _inputs(gen, gpu_device, dtype, (B, H, S, D), (B, H, S, D), D, True, torch.float32)
    table = oat.omni_rotary_table(rot, S, device=gpu_device)
    positions = torch.arange(S, device=gpu_device, dtype=torch.int32)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    y = oat.omni_qk_rotary(q, k, positions, table, wq, wk, EPS, interleaved)
    u = [torch.randn(q.shape, generator=gen).to(device=gpu_device, dtype=dtype) for _ in range(2)]
    grads = torch.autograd.grad(list(y), leaves, u)
    z = [torch.randn(t.shape, generator=gen).to(gpu_device).double() for t in leaves]
    angles = table[positions.long()]

    def loss(t):
        x = [leaf.detach().double() + t * d for leaf, d in zip(leaves, z)]
        return sum((norm_rotate(x[i], x[2 + i], angles, EPS, interleaved)[0] * u[i].double()).sum() for i in range(2))

    step = 1e-5
    slope = ((loss(step) - loss(-step)) / (2 * step)).item()
    got = sum((g.double() * d).sum() for g, d in zip(grads, z)).item()
    # every element of a 16-bit gradient is off by half a step at most (weights' gradients are fp32); differences: t^2
    room = sum((g.double().abs() * d.abs()).sum() for g, d in zip(grads[:2], z)).item() * half_step(dtype) * 1.1 + 1e-3
    assert abs(slope - got) <= room, (slope, got, room)


@pytest.mark.parametrize("layout", ["bshd", "packed", "fused", "odd_stride", "misaligned", "expanded"])
def test_layouts(gpu_device, layout):
    gen = torch.Generator().manual_seed(11)
    dtype, B, S, Hq, Hk, D = torch.bfloat16, 2, 37, 6, 2, 64
    table = oat.omni_rotary_table(D, S, device=gpu_device)
    positions = torch.arange(S, device=gpu_device)
    make = lambda *shape: torch.randn(shape, generator=gen).to(device=gpu_device, dtype=dtype)
    if layout == "packed":
        q, k = make(S, Hq, D), make(S, Hk, D)
        angles = table.unsqueeze(1)
    else:
        angles = table
        if layout == "bshd":
            q, k = make(B, S, Hq, D).transpose(1, 2), make(B, S, Hk, D).transpose(1, 2)
        elif layout == "fused":
            both = make(B, S, Hq + 2 * Hk, D).transpose(1, 2)
            q, k = both[:, :Hq], both[:, Hq:Hq + Hk]
        elif layout == "odd_stride":
            q, k = make(B, Hq, S, D + 3)[..., :D], make(B, Hk, S, D + 4)[..., 4:]
        elif layout == "misaligned":
            q, k = make(B * Hq * S * D + 1)[1:].view(B, Hq, S, D), make(B * Hk * S * D + 4)[4:].view(B, Hk, S, D)
        else:
            q, k = make(1, 1, S, D).expand(B, Hq, S, D), make(B, Hk, 1, D).expand(B, Hk, S, D)
    yq, yk = oat.omni_qk_rotary(q, k, positions, table)
    for got, x in ((yq, q), (yk, k)):
        _check(got, x, None, angles, False, dtype, layout)
    if layout == "bshd":
        assert yq.stride() == q.stride() and yk.stride() == k.stride()


def test_positions_weights_and_rounding_once(gpu_device):
    """int32 and int64 positions, one row for all batch elements or one each, shared positions (an image's tokens), those
    outside the table; fp32 weights; one side without a norm."""
    gen = torch.Generator().manual_seed(3)
    dtype, B, S, H, D = torch.float16, 3, 10, 4, 32
    q, k, wq, _ = _inputs(gen, gpu_device, dtype, (B, H, S, D), (B, H, S, D), D, True, torch.float32)
    table = oat.omni_rotary_table(16, 8, device=gpu_device)
    for positions in (torch.tensor([0, 1, 2, 2, 2, 2, 3, 7, 100, -4]), torch.randint(-3, 12, (B, S), generator=gen)):
        cut = positions.clamp(0, 7).to(gpu_device)
        angles = table[cut] if positions.dim() == 1 else table[cut].unsqueeze(1)
        for kind in (torch.int32, torch.int64):
            yq, yk = oat.omni_qk_rotary(q, k, positions.to(device=gpu_device, dtype=kind), table, query_norm=wq, eps=EPS)
            _check(yq, q, wq, angles, False, dtype, "normed")
            _check(yk, k, None, angles, False, dtype, "not normed")


def test_one_output_unused_and_frozen_weights(gpu_device):
    gen = torch.Generator().manual_seed(4)
    dtype, S, H, D = torch.bfloat16, 12, 2, 64
    q, k, wq, wk = _inputs(gen, gpu_device, dtype, (S, H, D), (S, H, D), D, True)
    table = oat.omni_rotary_table(D, S, device=gpu_device)
    positions = torch.arange(S, device=gpu_device)
    q.requires_grad_()
    wq.requires_grad_()
    yq, yk = oat.omni_qk_rotary(q, k, positions, table, wq, wk, EPS)
    both = torch.autograd.grad(yq.float().sum() + 0 * yk.float().sum(), [q, wq], retain_graph=True)
    alone = torch.autograd.grad(yq.float().sum(), [q, wq])
    for a, b in zip(both, alone):
        assert torch.equal(a, b)
    k.requires_grad_()
    yq, yk = oat.omni_qk_rotary(q, k, positions, table, wq, wk, EPS)
    with pytest.raises(RuntimeError, match="gradients of its gradients"):
        torch.autograd.grad(yk.float().sum(), k, create_graph=True)


def test_same_bits_every_time_and_in_a_graph(gpu_device):
    gen = torch.Generator().manual_seed(6)
    dtype, B, S, Hq, Hk, D = torch.bfloat16, 2, 300, 8, 2, 128
    q, k, wq, wk = _inputs(gen, gpu_device, dtype, (B, Hq, S, D), (B, Hk, S, D), D, True)
    dyq, dyk = torch.randn_like(q), torch.randn_like(k)
    table = oat.omni_rotary_table(D, S, device=gpu_device)
    positions = torch.arange(S, device=gpu_device)
    static = [t.clone() for t in (q, k, wq, wk, dyq, dyk)]

    def step(q, k, wq, wk, dyq, dyk):
        leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        y = oat.omni_qk_rotary(*leaves[:2], positions, table, *leaves[2:], EPS)
        return [t.detach() for t in y] + list(torch.autograd.grad(list(y), leaves, [dyq, dyk]))

    first = step(*static)
    for a, b in zip(first, step(*static)):
        assert torch.equal(a, b)
    side = torch.cuda.Stream(device=gpu_device)
    side.wait_stream(torch.cuda.current_stream(gpu_device))
    with torch.cuda.stream(side):
        step(*static)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = step(*static)
    torch.cuda.synchronize()
    for rep in range(3):
        for t in static:
            t.copy_(torch.randn(t.shape, generator=gen).to(t.dtype))
        eager = [t.clone() for t in step(*static)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b), f"replay {rep}"


def test_empty_and_large_offsets(gpu_device):
    table = oat.omni_rotary_table(64, 4, device=gpu_device)
    q = torch.zeros(0, 4, 64, dtype=torch.float16, device=gpu_device, requires_grad=True)
    w = torch.ones(64, dtype=torch.float16, device=gpu_device, requires_grad=True)
    yq, yk = oat.omni_qk_rotary(q, q, torch.zeros(0, dtype=torch.int64, device=gpu_device), table, w, w)
    assert yq.shape == q.shape
    gq, gw = torch.autograd.grad(yq.sum() + yk.sum(), [q, w])
    assert gq.shape == q.shape and bool((gw == 0).all())
    # an operand whose last rows lie beyond 2^31 elements
    big = torch.zeros(2, 1, 2, 1 << 30, dtype=torch.float16, device=gpu_device)
    gen = torch.Generator().manual_seed(9)
    x = torch.randn(2, 1, 2, 64, generator=gen).to(device=gpu_device, dtype=torch.float16)
    big[..., :64] = x
    yq, yk = oat.omni_qk_rotary(big[..., :64], x, torch.tensor([1, 3], device=gpu_device), table)
    assert torch.equal(yq, yk)
