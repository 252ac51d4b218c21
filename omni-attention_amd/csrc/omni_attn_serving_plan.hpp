// How a launch of the packed-sequence attention is cut into units, from what the host knows: tokens, sequences, heads
// (the lengths are on the device).  (Nothing here needs a GPU compiler.)
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace omni_attn {

struct ServePlan {
  bool tiles;      // tiles of 128 rows and four waves; else 32 rows and a wave of its own
  float share;     // units per key head that the steps are shared over, 0: whole tiles
  int64_t units;   // units per key head that there is a place for
  int rows() const { return tiles ? 128 : 32; }
  size_t workspace_bytes(int Hk, int D) const {
    return share == 0.f ? 0 : size_t(units) * size_t(Hk) * size_t(rows()) * size_t(D + 2) * sizeof(float);
  }
};

// T tokens in B sequences, Hk key heads with G query heads each; cus: compute units.
inline ServePlan plan_serve(int64_t T, int64_t B, int Hk, int G, bool paged, int cus) {
  ServePlan s;
  s.tiles = T * G > 64 * B;
  const int64_t slots = int64_t(cus) * (s.tiles ? 2 : 5);
  // tiles of all sequences, at most: each has one that is not full
  const int64_t tiles = T * G / s.rows() + B;
  const int64_t wanted = s.tiles ? slots : 2 * slots;
  const bool parts = s.tiles ? tiles * Hk < slots : (paged || tiles * Hk < wanted);
  s.share = parts ? float((wanted + Hk - 1) / Hk) : 0.f;
  // (the sum of what every tile is over a whole number of parts; one more workgroup, so that there is always one
  // without a unit, which clears rows behind the last sequence)
  s.units = tiles + 1 + (parts ? int64_t(s.share) + 1 : 0);
  return s;
}

// Workgroups, so that every key head has `units` of them (the dealing gives XCDs whole heads, or heads whole XCDs).
inline int64_t serve_blocks(int64_t units, int Hk, int n_xcd) {
  if (Hk % n_xcd != 0 && n_xcd % Hk == 0) {
    const int per = n_xcd / Hk;
    return (units + per - 1) / per * n_xcd;
  }
  return units * Hk;
}

}  // namespace omni_attn
