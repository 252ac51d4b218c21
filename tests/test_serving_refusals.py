"""What the rotation, the cache and the packed attention refuse, before anything is launched (CPU), and the tables of
cosines and sines against their definition."""
import ctypes
import math
import os
import random
import subprocess

import pytest
import torch

import omni_attn_capi
import omni_attn_torch as oat

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "omni-attention_amd", "csrc")


class Strides(ctypes.Structure):
    _fields_ = [("batch", ctypes.c_int64), ("head", ctypes.c_int64), ("row", ctypes.c_int64)]


ONE = ctypes.c_void_p(4096)  # any non-null address: checks come first
NULL = ctypes.c_void_p(0)
AT = Strides(0, 128, 1024)


def test_operators_refuse_tensors_of_the_wrong_kind():
    q = torch.zeros(4, 2, 64, dtype=torch.float16)
    i = torch.zeros(4, dtype=torch.int32)
    pages = torch.zeros(2, 2, 16, 64, dtype=torch.float16)
    table = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="GPU tensor"):
        oat.omni_qk_rotary(q, q, i, table)
    with pytest.raises(ValueError, match="GPU tensor"):
        oat.omni_cache_append(q, q, pages, pages, i.view(1, 4), i[:1], i[:2])
    with pytest.raises(ValueError, match="GPU tensor"):
        oat.omni_attention_packed(q, q, q, i[:2])
    with pytest.raises(ValueError, match="GPU tensor"):
        oat.omni_attention_paged(q, pages, pages, i.view(1, 4), i[:1], i[:2])


def test_rotary_codes():
    lib = omni_attn_capi.load_library()
    f = lib.omni_attn_qk_rotary_gfx950

    def call(q=ONE, at=AT, table=ONE, wq=NULL, B=1, S=2, Hq=2, Hk=1, D=64, rot=64, rows=8, eps=1e-6, dtype=1):
        return f(q, ONE, at, AT, ONE, ONE, AT, AT, table, ONE, ctypes.c_int64(0), 0, wq, NULL, 0, B, S, Hq, Hk, D, rot, rows,
                 ctypes.c_float(eps), 0, dtype, NULL)

    assert call(q=NULL) == 1 and call(table=NULL) == 1
    for bad in (dict(B=0), dict(S=0), dict(Hq=0), dict(Hk=0), dict(rot=12), dict(rot=72), dict(rows=0), dict(eps=-1.0),
                dict(eps=float("nan")), dict(eps=float("inf"))):
        assert call(**bad) == 2, bad
    assert call(D=260) == 3 and call(D=60) == 3 and call(D=0) == 3
    assert call(dtype=2) == 5
    assert call(q=ctypes.c_void_p(4100)) == 8 and call(at=Strides(0, 126, 1024)) == 8 and call(table=ctypes.c_void_p(4100)) == 8
    assert call(wq=ctypes.c_void_p(4104)) == 8
    assert call(at=Strides(0, 128, 1 << 40)) == 7
    b = lib.omni_attn_qk_rotary_bwd_gfx950

    def back(q=ONE, wq=ONE, dwq=ONE, ws=ONE, size=1 << 30):
        return b(ONE, ONE, q, ONE, AT, AT, AT, AT, ONE, ONE, AT, AT, dwq, NULL, ONE, ONE, ctypes.c_int64(0), 0, wq, NULL, 0, ws,
                 ctypes.c_size_t(size), 1, 2, 2, 1, 64, 64, 8, ctypes.c_float(0), 0, 1, NULL)

    assert back(q=NULL) == 1 and back(wq=NULL) == 1
    assert back(ws=NULL) == 9 and back(size=16) == 9
    lib.omni_attn_qk_rotary_bwd_workspace_bytes.restype = ctypes.c_size_t
    size = lib.omni_attn_qk_rotary_bwd_workspace_bytes
    assert size(0, 1, 64) == 0 and size(1, 1, 64) == 512 and size(1, 1 << 20, 64) == size(1, 1 << 30, 64)


def test_append_codes():
    f = omni_attn_capi.load_library().omni_attn_cache_append_gfx950

    def call(q=NULL, qo=NULL, k=ONE, pages=ONE, table=ONE, tokens=1, seqs=1, Hq=0, Hk=1, D=64, num=1, page=16, width=1, rot=64):
        return f(q, k, ONE, AT, AT, AT, qo, AT, pages, ONE, ONE, ONE, ONE, table, NULL, 0, NULL, NULL, 0, tokens, seqs, Hq, Hk, D,
                 num, page, width, rot, 8, ctypes.c_float(0), 0, 1, NULL)

    assert call(k=NULL) == 1 and call(pages=NULL) == 1 and call(table=NULL) == 1 and call(q=ONE) == 1
    for bad in (dict(tokens=0), dict(seqs=0), dict(num=0), dict(page=0), dict(page=24), dict(width=0), dict(Hq=2), dict(Hk=0),
                dict(rot=20)):
        assert call(**bad) == 2, bad
    assert call(D=7) == 3
    assert call(k=ctypes.c_void_p(4100)) == 8 and call(pages=ctypes.c_void_p(4100)) == 8


def test_attention_codes():
    lib = omni_attn_capi.load_library()

    def packed(q=ONE, at=AT, T=4, B=1, Hq=4, Hk=2, D=64, dtype=0, cap=0.0):
        return lib.omni_attn_packed_gfx950(q, ONE, ONE, at, AT, AT, ONE, NULL, ONE, NULL, ctypes.c_size_t(0), T, B, Hq, Hk, D, 1,
                                           dtype, ctypes.c_float(cap), NULL)

    def paged(q=ONE, table=ONE, D=64, num=1, page=16, width=1, Hq=4, T=4, cap=0.0):
        return lib.omni_attn_paged_gfx950(q, AT, ONE, ONE, ONE, NULL, table, ONE, ONE, NULL, ctypes.c_size_t(0), T, 1, Hq, 2, D,
                                          num, page, width, 1, 0, ctypes.c_float(cap), NULL)

    assert packed(q=NULL) == 1 and paged(q=NULL) == 1 and paged(table=NULL) == 1
    for bad in (dict(T=0), dict(B=0), dict(Hq=3), dict(Hk=0), dict(cap=-1.0), dict(cap=float("nan")), dict(cap=float("inf"))):
        assert packed(**bad) == 2, bad
    for bad in (dict(num=0), dict(page=8), dict(page=48), dict(page=1 << 17), dict(width=0), dict(Hq=5)):
        assert paged(**bad) == 2, bad
    assert packed(D=96) == 3 and paged(D=256) == 3
    assert packed(dtype=3) == 5
    assert packed(T=1 << 29) == 7 and packed(T=1, Hq=1 << 18) == 7 and paged(width=1 << 27) == 7 and packed(at=Strides(0, 128, 1 << 30)) == 7
    assert packed(q=ctypes.c_void_p(4104)) == 8 and packed(at=Strides(0, 124, 1024)) == 8


def test_packed_backward_codes():
    lib = omni_attn_capi.load_library()
    f = lib.omni_attn_packed_bwd_gfx950

    def call(q=ONE, dq=ONE, lse=ONE, at=AT, ws=ONE, size=1 << 20, T=4, B=1, Hq=4, Hk=2, D=64, dtype=0, cap=0.0):
        return f(q, ONE, ONE, ONE, ONE, lse, at, AT, AT, AT, dq, ONE, ONE, ONE, ws, ctypes.c_size_t(size), T, B, Hq, Hk, D, 1, dtype,
                 ctypes.c_float(cap), NULL)

    assert call(q=NULL) == 1 and call(dq=NULL) == 1 and call(lse=NULL) == 1
    for bad in (dict(T=0), dict(B=0), dict(Hq=3), dict(cap=-1.0), dict(cap=float("nan"))):
        assert call(**bad) == 2, bad
    assert call(D=96) == 3 and call(dtype=2) == 5
    assert call(at=Strides(0, 128, 1 << 25)) == 7 and call(at=Strides(0, 1 << 30, 1024)) == 7
    assert call(dq=ctypes.c_void_p(4104)) == 8 and call(at=Strides(0, 124, 1024)) == 8
    assert call(ws=NULL) == 9 and call(size=60) == 9
    lib.omni_attn_packed_bwd_workspace_bytes.restype = ctypes.c_size_t
    assert lib.omni_attn_packed_bwd_workspace_bytes(4, 4) == 64 and lib.omni_attn_packed_bwd_workspace_bytes(0, 4) == 0


@pytest.mark.parametrize("rot,scaling,factor", [(64, None, 1.0), (8, "linear", 4.0), (128, "ntk", 8.0), (128, "yarn", 16.0), (32, "yarn", 1.0)])
def test_rotary_table(rot, scaling, factor):
    theta, rows, original = 10000.0, 300, 64
    got = oat.omni_rotary_table(rot, rows, theta, scaling, factor, original, device="cpu")
    assert got.shape == (rows, rot) and got.dtype == torch.float32
    base = theta * factor ** (rot / (rot - 2)) if scaling == "ntk" else theta
    scale = 0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0
    for position in (0, 1, 63, 299):
        for i in range(rot // 2):
            turn = base ** (-2 * i / rot)
            if scaling == "linear":
                turn /= factor
            if scaling == "yarn":
                # turns over the original positions: more than 32 stay, fewer than 1 are divided by the factor
                pair = lambda turns: rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
                low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), rot - 1)
                ramp = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
                turn = turn * (1 - ramp) + turn / factor * ramp
            # (a cosine is rounded to 32 bits once; its angle is worked out in 64 bits twice)
            assert abs(got[position, i].item() - scale * math.cos(position * turn)) <= 2.0 ** -24 * scale * 1.01
            assert abs(got[position, rot // 2 + i].item() - scale * math.sin(position * turn)) <= 2.0 ** -24 * scale * 1.01
    if scaling == "ntk":  # the slowest pair turns 1 / factor as far, the fastest as far as before
        plain = theta ** (-(rot - 2) / rot)
        assert math.isclose(base ** (-(rot - 2) / rot), plain / factor, rel_tol=1e-12)


def test_rotary_table_keeps_far_positions_and_refuses():
    far = oat.omni_rotary_table(8, 1 << 20, device="cpu")
    position = (1 << 20) - 1
    assert abs(far[position, 0].item() - math.cos(position)) <= 2.0 ** -24
    for bad in (dict(rotary_dim=0), dict(rotary_dim=7), dict(max_positions=0), dict(theta=1.0), dict(factor=0.5),
                dict(factor=float("inf")), dict(scaling="other"), dict(scaling="yarn"), dict(scaling="ntk", rotary_dim=2),
                dict(scaling="yarn", original_positions=64, beta_fast=1.0)):
        with pytest.raises(ValueError):
            oat.omni_rotary_table(**dict(dict(rotary_dim=16, max_positions=4, device="cpu"), **bad))


PROGRAM = r"""
#include "omni_attn_serving_plan.hpp"
#include <cmath>
#include <cstdio>
#include <vector>
using namespace omni_attn;
// What the kernels count on the device, over the sequences that come in: tokens, keys.
int main() {
  int B, Hk, G, capacity;
  while (scanf("%d %d %d %d", &B, &Hk, &G, &capacity) == 4) {
    std::vector<long long> n(B), kv(B);
    long long T = 0;
    for (int b = 0; b < B; ++b) {
      if (scanf("%lld %lld", &n[b], &kv[b]) != 2) return 1;
      T += n[b];
    }
    const ServePlan s = plan_serve(T, B, Hk, G, capacity, 256);
    const long long M = s.rows;
    long long units = 0, part = 0;
    if (s.share > 0.f) {
      float all = 0.f;
      for (int b = 0; b < B; ++b) all += float((n[b] * G + M - 1) / M) * float((kv[b] + 63) / 64);
      part = (long long)std::ceil(all / s.share);
      if (part < s.least_steps) part = s.least_steps;
    }
    for (int b = 0; b < B; ++b) {
      const long long steps = (kv[b] + 63) / 64;
      long long parts = part == 0 || steps <= part ? 1 : (steps + part - 1) / part;
      if (parts > 1) {  // as even as whole steps allow
        const long long each = (steps + parts - 1) / parts;
        parts = (steps + each - 1) / each;
      }
      units += (n[b] * G + M - 1) / M * parts;
    }
    long long at_head = 0;
    for (int xcds : {1, 8}) {  // every key head gets its units
      const long long blocks = serve_blocks(s.units, Hk, xcds);
      at_head = Hk % xcds == 0 ? blocks / Hk : (xcds % Hk == 0 ? blocks / xcds * (xcds / Hk) : blocks / Hk);
      if (at_head < s.units) at_head = -1;
      if (at_head < 0) break;
    }
    printf("%lld %lld %lld %d %d %d\n", units, (long long)s.units, at_head, int(s.share > 0.f), s.rows, s.waves);
  }
}
"""


def test_every_unit_has_a_place(tmp_path):
    """The workgroups and the workspace hold all units that the device finds, whatever the lengths, and with whole tiles one
    workgroup is left that clears the rows behind the last sequence."""
    (tmp_path / "plan.cpp").write_text(PROGRAM)
    exe = str(tmp_path / "plan")
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", CSRC, str(tmp_path / "plan.cpp"), "-o", exe], check=True)
    rng = random.Random(1)
    lines = []
    for _ in range(3000):
        B, Hk, G, paged = rng.choice([1, 2, 3, 17, 64, 65, 300]), rng.choice([1, 2, 3, 8, 16, 24]), rng.choice([1, 2, 3, 8]), rng.random() < 0.5
        most = int(math.exp(rng.uniform(0, math.log(3000))))
        n = [1] * B if rng.random() < 0.3 else [rng.randint(0, most) for _ in range(B)]
        kv = [m + rng.randint(0, int(math.exp(rng.uniform(0, 11)))) if paged else m for m in n]
        if sum(n) == 0:
            n[0] = kv[0] = 1
        capacity = max(kv) + rng.choice([0, 100, 10 ** 5]) if paged else 0
        lines.append(f"{B} {Hk} {G} {capacity} " + " ".join(f"{a} {b}" for a, b in zip(n, kv)))
    out = subprocess.run([exe], input="\n".join(lines), stdout=subprocess.PIPE, text=True, check=True).stdout.split("\n")
    assert len(out) == len(lines) + 1
    seen = set()
    for line, given in zip(out, lines):
        units, room, at_head, parts, rows, waves = map(int, line.split())
        seen.add((parts, rows, waves))
        assert units <= (room if parts else room - 1) and at_head >= room, given[:200]
    assert seen == {(0, 128, 4), (1, 128, 4), (0, 64, 4), (0, 32, 1), (0, 32, 4), (1, 32, 4)}
