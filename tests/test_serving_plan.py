"""What the kernels of packed sequences count and number on the device, on the CPU: units of batches whose offsets may be anything."""
import os
import random
import subprocess

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
