// How a launch of the packed-sequence attention is cut into units, from what the host knows: tokens, sequences, heads
// (the lengths are on the device).  (Nothing here needs a GPU compiler.)
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace omni_attn {

struct ServePlan {
  int rows;        // of a tile: 128, 64 or 32
  int waves;       // of a workgroup: 4, or 1 (tiles of 32 rows)
  float share;     // units per key head that the steps are shared over, 0: whole tiles
  int least_steps; // steps that a part may have in any case
  int places;      // units per key head that run at once, where tiles are shared (two workgroups to a compute unit)
  int64_t units;   // units per key head that there is a place for
  int64_t slots;   // parts per key head that there is a place for in the workspace (whole tiles need none)
  int64_t counted; // sequences whose units a kernel of its own counts, or 0
  // the parts' rows and statistics, four words per token, two per counted sequence and one more
  size_t workspace_bytes(int64_t T, int Hk, int D) const {
    if (share == 0.f) return 0;
    return size_t(slots) * size_t(Hk) * size_t(rows) * size_t(D + 2) * sizeof(float) + size_t(T) * 16 + size_t(counted) * 8 + 4;
  }
};

// Few sequences whose parts are weighed on the device instead of sharing the steps evenly, over a cache alone: at most so many.
constexpr int weighed_sequences(int rows) { return rows == 128 ? 16 : 8; }
// ... with `steps` steps in all tiles of a key head, which take more than two rounds of the units that run at once.
constexpr bool weighed(int64_t B, int rows, float steps, int places) { return B <= weighed_sequences(rows) && steps > 2.f * float(places); }

// T tokens in B sequences, Hk key heads with G query heads each; capacity: keys that a page table has room for, 0:
// packed; cus: compute units.  Lengths are not known here: a sequence is taken to have T / B tokens, and keys of a
// cache that there may be any number of.
inline ServePlan plan_serve(int64_t T, int64_t B, int Hk, int G, int64_t capacity, int cus) {
  ServePlan s;
  const int64_t all = T * G;
  s.rows = 32;
  s.waves = 4;
  const auto tiles_of = [&](int64_t M) { return all / M + B; };  // at most: every sequence has one that is not full
  const int64_t keys = capacity != 0 ? capacity : T / B;
  int64_t wanted = 0;  // units in all, where tiles are shared by parts
  s.least_steps = 2;
  if (all <= 64 * B) {
    // Single tokens, a few.  One wave per tile where keys are few and tiles more than the card holds at a time: D=128, 32 / 8
    // heads, 512 sequences of 30 - 100 keys 28 us, 46 with four waves, 52 with four waves and parts; 256 of 100 - 300 keys 37, 39
    // and 45; 200 prompts of 60 tokens, as many key heads, 24 and 41.  Else four waves and parts: 8 tokens after 60000 keys 343,
    // 616 with whole tiles, 2160 with one wave (8 after 2000 keys 26 us, 23 and 65, 64 after 500 - 1500 keys 51, 44 and 58: what
    // this loses by, lengths are not known here).  Twice as many units or half as many: within 3 %.
    if ((keys <= 512 && tiles_of(32) * Hk > 4 * cus) || (capacity == 0 && keys <= 128)) s.waves = 1;
    if (s.waves == 4 && keys > 512) wanted = 4 * cus;
    s.least_steps = 4;
  } else if (tiles_of(32) * Hk <= 2 * cus + B * Hk && keys <= 2560) {
    // Prompts whose 32-row tiles all run at once: four waves on the keys of each.  512 tokens, D=64, 8 heads 6.8 us, 10.4 with
    // tiles of 128 rows; 2048 tokens 15 and 26; D=128, 32 / 8 heads, 512 tokens 11.2 and 13.5 (1024 tokens, beyond the line,
    // 26 and 22; 8192 tokens, 2 heads, 81 and 63 in parts).
  } else {
    // Parts where the tiles leave compute units without work: 4096 tokens, one head, 26 us, 61 whole; 8192, 2 heads, 64 and
    // 117; 512 and 300 new tokens after 15000 and 7000, 32 / 8 heads, D=128, 188 and 307; 4096 after 10000, 8 heads, D=64, 132
    // and 156 (1500 after 6000, 32 / 8 heads, beyond the line, 198 and 170).
    s.rows = 128;
    if (tiles_of(128) * Hk <= (capacity != 0 ? 5 * cus / 4 : cus) && keys > 2560) wanted = 3 * cus;
    // Tiles of 64 rows and two groups of waves where there are fewer tiles of 128 than the card holds at a time, and their
    // walks are not short: 9 prompts of 35 - 1047 tokens, D=64, 16 heads, capped scores 20 us, 26 with 128 rows; 4 x 1157
    // tokens, 8 heads 23.6 and 27.5; 1024 tokens, D=128, 32 / 8 heads 19.3 and 22.1 (beyond the line: 2048 tokens 46.4 and
    // 44.7; 4 x 512 25.8 and 19.5; 16 x 100 tokens, D=64, 16 heads 8.2 and 7.6).
    if (wanted == 0 && (2 * all / 128 + B) * Hk <= 7 * cus / 2 && keys >= 256 && keys <= 2560) s.rows = 64;
    s.least_steps = 8;
  }
  const int64_t tiles = tiles_of(s.rows);
  const bool parts = wanted != 0;
  s.counted = parts && B > 64 ? B : 0;
  s.share = parts ? float((wanted + Hk - 1) / Hk) : 0.f;
  // (the sum of what every tile is over a whole number of parts; one more workgroup, so that there is always one
  // without a unit, which clears rows behind the last sequence)
  s.places = 2 * cus >= Hk ? 2 * cus / Hk : 1;
  s.units = tiles + 1 + (parts ? int64_t(s.share) + 1 : 0);
  if (parts && s.rows == 128) s.units += 3 * s.places / 2;  // (three rounds of them)
  // A tile is cut where it has more steps than a part, so it has less than twice its steps over a part's, and all parts
  // together are less than twice the share: however many sequences there are.  (1024 single tokens, 32 / 8 heads, D=128: 34 MB for
  // 153 with a place for every tile; 4096, 32 / 32 heads, 35 MB for 2.2 GB.)  Weighed parts are as many as there are units.
  s.slots = !parts ? 0 : (B <= weighed_sequences(s.rows) || s.units < 2 * int64_t(s.share) + 2 ? s.units : 2 * int64_t(s.share) + 2);
  return s;
}

// Tile number of unit `rank` of a sequence whose units start at number `first`: the last tile comes first.  -1: the unit is not
// one of its tiles.  (Offsets that run backwards make a search over their sequences' first units end anywhere, before a
// sequence's units too: an empty one has no tile then either.)
constexpr int whole_tile(int rank, int first, int tiles) { return rank < first || rank - first >= tiles ? -1 : tiles - 1 - (rank - first); }

// Workgroups, so that every key head has `units` of them (the dealing gives XCDs whole heads, or heads whole XCDs).
inline int64_t serve_blocks(int64_t units, int Hk, int n_xcd) {
  if (Hk % n_xcd != 0 && n_xcd % Hk == 0) {
    const int per = n_xcd / Hk;
    return (units + per - 1) / per * n_xcd;
  }
  return units * Hk;
}

}  // namespace omni_attn
