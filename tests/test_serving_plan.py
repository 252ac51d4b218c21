"""What the kernels of packed sequences count and number on the device, on the CPU: units of batches whose offsets may be
anything, places of parts, and which batches' parts are weighed."""
import math
import os
import random
import subprocess

import pytest
import torch

from serving_weighed import CHUNKS, FEW, bound, make, reference

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "omni-attention_amd", "csrc")


def _run(tmp_path, program, lines):
    (tmp_path / "plan.cpp").write_text(program)
    exe = str(tmp_path / "plan")
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", CSRC, str(tmp_path / "plan.cpp"), "-o", exe], check=True)
    return subprocess.run([exe], input="\n".join(lines), stdout=subprocess.PIPE, text=True, check=True).stdout.split("\n")[:-1]


# The search over more than 64 sequences as a wave makes it: 64 first units are looked at in a round.
SEARCH = r"""
#include "omni_attn_serving_plan.hpp"
#include <cstdio>
#include <vector>
int main() {
  int B, T, G, M;
  while (scanf("%d %d %d %d", &B, &T, &G, &M) == 4) {
    std::vector<int> cu(B + 1);
    for (int& x : cu)
      if (scanf("%d", &x) != 1) return 1;
    auto cut = [&](int x) { return x < 0 ? 0 : (x > T ? T : x); };
    auto start = [&](int b) { return int((long long)(b == 0 ? 0 : cut(cu[b])) * G / M) + b; };
    long long outside = 0, found = 0, all = 0;
    std::vector<int> tiles(B);
    for (int b = 0; b < B; ++b) {
      const int from = b == 0 ? 0 : cut(cu[b]), to = cu[b + 1] < from ? from : cut(cu[b + 1]);
      tiles[b] = int(((long long)(to - from) * G + M - 1) / M);
      all += tiles[b];
    }
    for (int rank = 0; rank < int((long long)T * G / M) + B + 1; ++rank) {
      int count = 0;
      for (int left = B; left > 0;) {
        const int step = (left + 63) / 64;
        int passed = 0;
        for (int lane = 0; lane < 64; ++lane) {
          const int i = (lane + 1) * step;
          passed += i <= left && start(count + i) <= rank ? step : 0;
        }
        count += passed;
        left = left - passed < step - 1 ? left - passed : step - 1;
      }
      if (count == B) continue;
      const int tile = omni_attn::whole_tile(rank, start(count), tiles[count]);
      found += tile >= 0;
      outside += tile >= tiles[count];
    }
    printf("%lld %lld %lld\n", outside, found, all);
  }
}
"""


def test_units_of_offsets_that_run_backwards(tmp_path):
    """No unit lies outside its sequence, whatever the offsets (the tile of an empty sequence has no row to read); of offsets that
    do not decrease every tile is found once."""
    rng = random.Random(1)
    lines, ordered = [], []
    for i in range(200):
        B, T, G, M = rng.choice([65, 70, 130, 300]), rng.choice([200, 1000, 5000]), rng.choice([1, 4, 8]), rng.choice([32, 64, 128])
        cu = [0] + [rng.randint(-5, T + 5) if rng.random() < 0.2 else rng.choice([0, T // 2]) for _ in range(B)]
        ordered.append(i % 2 == 0)
        if ordered[-1]:
            cu = sorted(max(0, min(x, T)) for x in cu)
        lines.append(f"{B} {T} {G} {M} " + " ".join(map(str, cu)))
    got = [tuple(map(int, line.split())) for line in _run(tmp_path, SEARCH, lines)]
    assert len(got) == len(lines)
    for (outside, found, tiles), in_order in zip(got, ordered):
        assert outside == 0
        if in_order:
            assert found == tiles


# What a launch in parts needs: parts of cut tiles as the device numbers them, and the places that the plan has for them.
PARTS = r"""
#include "omni_attn_serving_plan.hpp"
#include <cmath>
#include <cstdio>
#include <vector>
int main() {
  int B, Hk, G, D, capacity;
  while (scanf("%d %d %d %d %d", &B, &Hk, &G, &D, &capacity) == 5) {
    std::vector<long long> n(B), kv(B);
    long long T = 0;
    for (int b = 0; b < B; ++b) {
      if (scanf("%lld %lld", &n[b], &kv[b]) != 2) return 1;
      T += n[b];
    }
    const omni_attn::ServePlan s = omni_attn::plan_serve(T, B, Hk, G, capacity, 256);
    const long long M = s.rows;
    long long cut = 0, most = 0;
    if (s.share > 0.f) {
      float all = 0.f;
      for (int b = 0; b < B; ++b) all += float((n[b] * G + M - 1) / M) * float((kv[b] + 63) / 64);
      most = (long long)std::ceil(all / s.share);
      if (most < s.least_steps) most = s.least_steps;
      for (int b = 0; b < B; ++b) {
        const long long steps = (kv[b] + 63) / 64;
        if (steps <= most) continue;
        const long long parts = (steps + most - 1) / most, each = (steps + parts - 1) / parts;
        cut += (n[b] * G + M - 1) / M * ((steps + each - 1) / each);
      }
    }
    printf("%d %lld %lld %zu\n", s.share > 0.f, cut, (long long)s.slots, s.workspace_bytes(T, Hk, D));
  }
}
"""


def test_workspace_holds_the_parts_and_not_the_batch(tmp_path):
    """Every part has a place, and the workspace does not grow with the number of sequences, but for the words that each has."""
    rng = random.Random(2)
    cases = []
    for _ in range(2000):
        B, Hk, G = rng.choice([1, 5, 9, 17, 64, 65, 300, 2000]), rng.choice([1, 2, 8, 24, 32]), rng.choice([1, 2, 4, 8])
        n = [1] * B if rng.random() < 0.7 else [rng.randint(0, rng.choice([3, 40, 400])) for _ in range(B)]
        n[0] = max(n[0], 1)
        long = rng.choice([1, 3, 10])
        kv = [m + (rng.randint(2000, 60000) if rng.randrange(B) < long else rng.randint(0, rng.choice([10, 2000]))) for m in n]
        cases.append((B, Hk, G, rng.choice([32, 64, 128]), max(kv) + rng.choice([0, 10 ** 5]), n, kv))
    for B, Hk, G in ((1024, 8, 4), (4096, 8, 4), (4096, 32, 1), (20000, 1, 1)):
        cases.append((B, Hk, G, 128, 1 << 17, [1] * B, [500 + b % 500 for b in range(B)]))
    got = _run(tmp_path, PARTS, [f"{B} {Hk} {G} {D} {c} " + " ".join(f"{a} {b}" for a, b in zip(n, kv)) for B, Hk, G, D, c, n, kv in cases])
    assert len(got) == len(cases)
    seen = 0
    for line, (B, _, _, _, _, n, _) in zip(got, cases):
        parts, cut, slots, size = map(int, line.split())
        seen += parts
        assert cut <= slots and size <= 16 * sum(n) + 8 * B + 4 + 128 * 2 ** 20
    assert seen > 500


WEIGHED = r"""
#include "omni_attn_serving_plan.hpp"
#include <cstdio>
int main() {
  int B, Hk, G, capacity;
  while (scanf("%d %d %d %d", &B, &Hk, &G, &capacity) == 4) {
    long long T = 0, n[64], kv[64];
    for (int b = 0; b < B; ++b) {
      if (scanf("%lld %lld", n + b, kv + b) != 2) return 1;
      T += n[b];
    }
    const omni_attn::ServePlan s = omni_attn::plan_serve(T, B, Hk, G, capacity, 256);
    float all = 0.f;
    for (int b = 0; b < B; ++b) all += float((n[b] * G + s.rows - 1) / s.rows) * float((kv[b] + 63) / 64);
    printf("%d %d %d\n", s.rows, s.waves, int(s.share > 0.f && omni_attn::weighed(B, s.rows, all, s.places)));
  }
}
"""


def test_the_weighed_batches_are_weighed(tmp_path):
    """The batches that stand for weighed parts take that path on a card of 256 compute units: the single tokens and a few in
    tiles of 32 rows, the chunks in tiles of 128."""
    lines = []
    for lens, cached, Hq, Hk, _ in FEW + CHUNKS:
        total = [n + c for n, c in zip(lens, cached)]
        lines.append(f"{len(lens)} {Hk} {Hq // Hk} {max(total)} " + " ".join(f"{n} {m}" for n, m in zip(lens, total)))
    got = [tuple(map(int, x.split())) for x in _run(tmp_path, WEIGHED, lines)]
    assert got == [(32, 4, 1)] * len(FEW) + [(128, 4, 1)] * len(CHUNKS)


@pytest.mark.parametrize("case", range(len(FEW) + len(CHUNKS)))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_bound_of_the_weighed_batches_tells_results_from_none(case, dtype):
    """An output of zeros, and one that leaves an eighth of the keys out, is beyond the bound in most elements."""
    lens, cached, Hq, Hk, D = (FEW + CHUNKS)[case]
    q, rows = make(torch.Generator().manual_seed(case), lens, cached, Hq, Hk, D, dtype)
    b = max(range(len(lens)), key=lambda i: cached[i] * (lens[i] > 0))
    at = sum(lens[:b])
    k, v = rows[b]
    q = q[at:at + lens[b]][-2:, :Hq // Hk]  # the sequence's last rows, one key head
    k, v = k[:, :1], v[:, :1]
    first = k.shape[0] - q.shape[0]
    want, mean, _, spread = reference(q, k, v, first, True)
    smax = (q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()).item() / math.sqrt(D)
    room = bound(want, mean, spread, dtype, D, smax)
    assert (want.abs() > room).double().mean().item() > 0.9
    cut = k.shape[0] // 8
    fewer = reference(q, k[cut:], v[cut:], first - cut, True)[0]
    assert ((fewer - want).abs() > room).double().mean().item() > 0.7  # (a fifth of the dimensions have no slope)
