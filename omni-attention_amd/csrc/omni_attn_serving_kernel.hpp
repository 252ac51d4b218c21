// Attention of packed sequences: new tokens of many sequences, one behind the other, over their own keys and
// values, which lie packed the same way or in the pages of a cache.  Query heads come in groups of G that share a
// key head.
//   O[t, h, :] = softmax_j( cap(Q[t, h, :] . K[j, h / G, :] / sqrt(D)) ) V[j, h / G, :]
// over the keys j of the token's sequence: those up to the token's own position, or all of them.  Sequence b has
// the tokens cu[b] .. cu[b + 1] - 1 and kv keys; its last token is at position kv - 1.
//
// As in the block-sparse forward everything is computed transposed, so that a lane owns one query row: S^T = K Q^T
// and O^T = V^T P^T with 32x32x16 matrix instructions, P in registers throughout.  A row here is a token and one of
// the G heads of a group: the rows of a tile share one key head, so K and V are read once for all of them, a single
// token fills G rows, and a tile of a prompt has few tokens, so little of its last steps is masked.
//
// Work is dealt on the device, because lengths are there: every workgroup finds the unit with its number.  A unit is a
// tile of rows and a range of keys (all of them, or where there are fewer units than the card holds, parts that are equal
// over the whole batch).  Parts leave their sums and maxima in a workspace, and a second kernel joins them.
#pragma once

#include "omni_attn_fwd_kernel.hpp"
#include "omni_attn_serving_plan.hpp"

namespace omni_attn {

// Where keys and values lie: packed, in pages of which a step of the walk reads one, or in smaller ones.  (A page looked up
// once a step, and not once a load: 8192 tokens, 32 / 8 heads, D=128, 490 us for 532, as fast as packed ones.)
enum Keys { kPacked, kPages, kSmallPages };
constexpr int kPageOfStep = 64;  // keys

struct ServeParams {
  const uint16_t* q;  // [T, Hk * G, D] at q_row, q_head
  const uint16_t* k;  // packed [T, Hk, D] at their strides, or pages [num_pages, Hk, page, D]
  const uint16_t* v;
  int64_t q_row, q_head;
  RowStrides k_at, v_at;  // (h, row) of packed keys and values
  uint16_t* o;            // [T, Hk * G, D]
  float* lse;             // [T, Hk * G] or null
  const int32_t* cu;      // [B + 1]
  const int32_t* kv_lens;     // [B]; null: packed
  const int32_t* page_table;  // [B, max_pages]
  int num_pages, max_pages, page_shift;
  int B, T, Hk, G;
  FastDiv group;       // by G
  FastDiv heads;       // by Hk
  int n_xcd;
  int causal;
  float share;         // units per key head that the batch's steps are shared over; 0: whole tiles
  int least_steps;     // ... and the steps that a part may have in any case
  int places;          // units per key head that run at once, where tiles are shared
  int units;           // units per key head that there is a place for
  int slots;           // parts per key head that there is a place for
  int32_t* ends;       // [2 B + 1] of batches that a kernel of its own counts: units up to and with each sequence; steps of a
                       // part; places of parts up to and with each sequence
  float* sums;         // [slots, Hk, M, D] unscaled O of parts
  float* stats;        // [slots, Hk, M, 2] their reference points (log2 domain) and sums of weights
  int32_t* joins;      // [T, 4] of a token: first token and number of parts of its sequence, place of its first part
  float sl2, softcap, cap_c2;
};

constexpr int kStepKeys = 64;  // lengths are counted in steps of as many keys

// Inclusive sum over the lanes before this one, and this one.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return x;
}
__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_zero(float x) {  // another lane's x, or 0 where there is none
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float wave_sum(float x) {
  x += dpp_zero<0x111, 0xf>(x);
  x += dpp_zero<0x112, 0xf>(x);
  x += dpp_zero<0x114, 0xf>(x);
  x += dpp_zero<0x118, 0xf>(x);
  x += dpp_zero<0x142, 0xa>(x);
  x += dpp_zero<0x143, 0xc>(x);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_max(int x) {
  const int y = __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
  return x > y ? x : y;
}
__device__ __forceinline__ int wave_max(int x) {
  x = dpp_max<0x118, 0xf>(dpp_max<0x114, 0xf>(dpp_max<0x112, 0xf>(dpp_max<0x111, 0xf>(x))));
  return __builtin_amdgcn_readlane(dpp_max<0x143, 0xc>(dpp_max<0x142, 0xa>(x)), 63);
}

struct Sequence {
  int first, n, kv;  // first token, tokens, keys
};
// (the first offset counts as 0; offsets that run backwards or beyond the tokens, and lengths beyond the page table, are
// cut)
__device__ __forceinline__ Sequence sequence_of(const ServeParams& p, int b) {
  Sequence s = {0, 0, 0};
  if (b < p.B) {
    int from = b == 0 ? 0 : p.cu[b], to = p.cu[b + 1];
    from = from < 0 ? 0 : (from > p.T ? p.T : from);
    to = to < from ? from : (to > p.T ? p.T : to);
    s.first = from;
    s.n = to - from;
    s.kv = s.n;
    if (p.kv_lens != nullptr) {
      const int64_t most = int64_t(p.max_pages) << p.page_shift;
      const int kv = p.kv_lens[b];
      s.kv = kv < 0 ? 0 : (kv > most ? int(most) : kv);
    }
  }
  return s;
}
template <int M>
__device__ __forceinline__ int tiles_of(const ServeParams& p, const Sequence& s) {
  return int((uint32_t(s.n) * uint32_t(p.G) + uint32_t(M - 1)) / uint32_t(M));
}
__device__ __forceinline__ int steps_of(int keys) { return (keys + kStepKeys - 1) / kStepKeys; }

__device__ __forceinline__ Sequence pick(const Sequence& s, int lane) {
  return {__builtin_amdgcn_readlane(s.first, lane), __builtin_amdgcn_readlane(s.n, lane), __builtin_amdgcn_readlane(s.kv, lane)};
}
// How many of at(1) .. at(n), which do not decrease, are at most `rank`: 64 of them are looked at in a round.
template <class F>
__device__ __forceinline__ int count_up_to(int n, int rank, int lane, F&& at) {
  int count = 0;
  for (int left = n; left > 0;) {
    const int step = (left + 63) / 64, i = (lane + 1) * step;
    const int passed = __builtin_popcountll(__builtin_amdgcn_ballot_w64(i <= left && at(i <= left ? count + i : n) <= rank)) * step;
    count += passed;
    left = left - passed < step - 1 ? left - passed : step - 1;
  }
  return count;
}

// A sequence's keys in parts of at most `most` steps: as few as that takes, as even as whole steps allow.
struct Parts {
  int n, steps;
};
__device__ __forceinline__ Parts parts_of(int kv, int most) {
  const int all = steps_of(kv);
  if (all <= most) return {1, all};
  const int n = int(uint32_t(all + most - 1) / uint32_t(most)), each = int(uint32_t(all + n - 1) / uint32_t(n));
  return {int(uint32_t(all + each - 1) / uint32_t(each)), each};
}
// The most steps of a part: the batch's steps (of all tiles) over the units that they are shared by.
__device__ __forceinline__ int part_steps(const ServeParams& p, float all) {
  const float steps = ceilf(all / p.share);
  const int part = steps < 1e9f ? int(steps) : 1000000000;
  return __builtin_amdgcn_readfirstlane(part < p.least_steps ? p.least_steps : part);
}

constexpr int kAll = 0x7fffffff;
// The same for a few sequences with many steps over a cache, which take long enough for their last round to count: the longest
// sequence is cut into 1, 2, ... (a multiple per lane), the others into parts that are no longer, and what ends first
// is taken: rounds of the units that run at once, each as long as a part and its start and end (about four steps).  Parts
// lie alike in all tiles of a sequence, so that these read the same keys at a time.  (100 new tokens after 20000 keys, 32 / 8
// heads, D=128: 60 us, 71 with the batch's steps over 1.5 times the units that run at once, 68 with even runs of steps that go
// on from tile to tile; 512 and 300 after 15000 and 7000: 202, 207, 209; 812 after 22000: 325, 347, 316; all three with a
// page looked up for every load, which left 58, 186 and 308 of the first.  Packed prompts,
// where causal tiles have fewer steps than are counted here: 8192 tokens, 2 heads, 72 us and 63 with the shares.  Single
// tokens: one after 60000 keys 63 us, 78 with the shares; 4 after 1000 - 8000 28 and 30.5; beyond the lines one after 4000
// 15.6 and 14.9, 16 after 300 - 16000 50 and 48.5, 60 after 4000 125 and 103.)
template <int M>
__device__ __forceinline__ int weighed_steps(const ServeParams& p, int tiles, int steps, int lane, int fallback) {
  constexpr int kEnds = 4;
  const int longest = wave_max(tiles > 0 ? steps : 0), all_tiles = wave_sum(tiles);
  if (longest <= p.least_steps) return fallback;
  const int stride = 1 + int(uint32_t(3 * p.places) / uint32_t(64 * (all_tiles < 1 ? 1 : all_tiles)));
  const int cut = (lane + 1) * stride;
  int most = int(uint32_t(longest + cut - 1) / uint32_t(cut));
  if (most < p.least_steps) most = p.least_steps;
  int units = 0;
  for (int b = 0; b < p.B; ++b) units += __builtin_amdgcn_readlane(tiles, b) * parts_of(__builtin_amdgcn_readlane(steps, b) * kStepKeys, most).n;
  const int rounds = int(uint32_t(units + p.places - 1) / uint32_t(p.places));
  // (the smallest time, and of the same the longest parts)
  const int time = units < p.units ? rounds * (most + kEnds) : 0x7fffffff;
  const int best = -wave_max(-time);
  if (best == 0x7fffffff) return fallback;
  return __builtin_amdgcn_readlane(most, __builtin_ctzll(__builtin_amdgcn_ballot_w64(time == best)));
}

struct Unit {
  Sequence seq;
  int b, tile;
  int step0, steps;  // range of steps (all that the tile has may be fewer)
  int base, slot;    // (shared by parts) place of the sequence's first part, and of this one
  int parts;         // parts of each of its tiles
  bool part;         // one of several: its sums are joined later
  bool found;        // no: (whole tiles) step0 is the number behind the last unit's (kAll: this number is left out)
};

// Unit number `rank` of tiles that are shared by parts: sequences in order, tiles in order, parts in order.  Up to 64
// sequences, one per lane, are counted by every wave (the same numbers in each: the same sums in the same order); more, by
// a kernel that goes before (512 single tokens after 500 - 1000 keys, 8 / 1 heads, D=128: 48 us, 54 with every wave counting
// eight per lane; 4096 of them, 32 / 8 heads, 2.1 ms and 5.7).
template <int M, bool WEIGH>
__device__ __forceinline__ Unit find_part(const ServeParams& p, int rank, int lane) {
  Sequence s;
  int b, most, in, base;
  if (p.ends != nullptr) {
    most = load_uniform(p.ends + p.B);
    b = count_up_to(p.B, rank, lane, [&](int i) { return p.ends[i - 1]; });
    if (b == p.B) return Unit{{}, 0, 0, 0, 0, 0, 0, 0, false, false};
    s = pick(sequence_of(p, b), 0);
    in = rank - (b == 0 ? 0 : load_uniform(p.ends + b - 1));
    base = b == 0 ? 0 : load_uniform(p.ends + p.B + b);
  } else {
    const Sequence own = sequence_of(p, lane);
    const int tiles = tiles_of<M>(p, own);
    const float all = wave_sum(float(tiles) * float(steps_of(own.kv)));
    most = part_steps(p, all);
    if (WEIGH && weighed(p.B, M, all, p.places)) most = weighed_steps<M>(p, tiles, steps_of(own.kv), lane, most);
    const int parts = parts_of(own.kv, most).n, mine = tiles * parts, end = wave_scan(mine);
    const int cut = parts > 1 ? mine : 0, cut_end = wave_scan(cut);
    const uint64_t beyond = __builtin_amdgcn_ballot_w64(end > rank);
    if (beyond == 0) return Unit{{}, 0, 0, 0, 0, 0, 0, 0, false, false};
    b = __builtin_ctzll(beyond);
    s = pick(own, b);
    in = rank - (__builtin_amdgcn_readlane(end, b) - __builtin_amdgcn_readlane(mine, b));
    base = __builtin_amdgcn_readlane(cut_end, b) - __builtin_amdgcn_readlane(cut, b);
  }
  const Parts parts = parts_of(s.kv, most);
  const int tile = int(uint32_t(in) / uint32_t(parts.n));
  // (counts of overlapping sequences, from offsets that run backwards, may pass 32 bits)
  if (in < 0 || tile >= tiles_of<M>(p, s) || (parts.n > 1 && (base < 0 || uint32_t(base) + uint32_t(in) >= uint32_t(p.slots))))
    return Unit{{}, 0, 0, 0, 0, 0, 0, 0, false, false};
  return Unit{s, b, tile, (in - tile * parts.n) * parts.steps, parts.steps, base, base + in, parts.n, parts.n > 1, true};
}

// Unit number `rank` of whole tiles.  Of up to 64 sequences those with most steps come first, so that a launch ends with
// short ones: steps are compared in sixteen levels, which four rounds of counting find.  One sequence, or more than 64, in
// order, the last tile of each first.  Their numbers need no counting: the tiles of sequence b start at number
// floor(cu[b] G / M) + b, which leaves room for all that the sequences before it can have, and out one number for some.
template <int M>
__device__ __forceinline__ Unit find_tile(const ServeParams& p, int rank, int lane) {
  constexpr int kLog = M == 128 ? 7 : (M == 64 ? 6 : 5);
  static_assert(M == 1 << kLog, "rows of a tile");
  if (p.B == 1 || p.B > 64) {
    const auto start = [&](int b) {
      int from = b == 0 ? 0 : p.cu[b];
      from = from < 0 ? 0 : (from > p.T ? p.T : from);
      return int(uint32_t(from) * uint32_t(p.G) >> kLog) + b;
    };
    const int b = count_up_to(p.B, rank, lane, start), first = __builtin_amdgcn_readfirstlane(start(b));
    if (b == p.B) return Unit{{}, 0, 0, first, 0, 0, 0, 1, false, false};
    const Sequence s = pick(sequence_of(p, b), 0);
    const int tile = whole_tile(rank, first, tiles_of<M>(p, s));
    return Unit{s, b, tile, tile < 0 ? kAll : 0, kAll, 0, 0, 1, false, tile >= 0};
  }
  const Sequence s = sequence_of(p, lane);
  const int most = wave_max(s.n > 0 ? steps_of(s.kv) : 0);
  int unit = 0;  // log2 of the steps of a level
  while ((most >> unit) > 15) ++unit;
  // tiles of a sequence with at least `steps` steps (its last ones)
  const int tiles = tiles_of<M>(p, s);
  auto long_tiles = [&](int steps) {
    if (steps <= 0) return tiles;
    if (!p.causal) return steps_of(s.kv) >= steps ? tiles : 0;
    const int token = kStepKeys * (steps - 1) - (s.kv - s.n);  // first token whose keys reach so far
    const int row = (token < s.n ? token : s.n) * p.G;
    return token >= s.n ? 0 : (token <= 0 ? tiles : tiles - (row >> kLog));
  };
  const int all = wave_sum(tiles);
  if (all <= rank) return Unit{{}, 0, 0, all, 0, 0, 0, 1, false, false};
  int level = 0, longer = 0;  // (tiles above the level)
  for (int bit = 8; bit != 0; bit >>= 1) {
    const int n = wave_sum(long_tiles((level | bit) << unit));
    if (n > rank) {
      level |= bit;
    } else {
      longer = n;
    }
  }
  const int from = long_tiles(level << unit), mine = from - (level == 15 ? 0 : long_tiles((level + 1) << unit));
  const int end = wave_scan(mine);
  rank -= longer;
  const uint64_t beyond = __builtin_amdgcn_ballot_w64(end > rank);
  const int at = beyond != 0 ? __builtin_ctzll(beyond) : 0;
  const int in = rank - (__builtin_amdgcn_readlane(end, at) - __builtin_amdgcn_readlane(mine, at));
  const int tile = __builtin_amdgcn_readlane(tiles - from + mine, at) - 1 - in;
  return Unit{pick(s, at), at, tile, 0, kAll, 0, 0, 1, false, true};
}
template <int M, bool WEIGH>
__device__ __forceinline__ Unit find_unit(const ServeParams& p, int rank, int lane) {
  return p.share > 0.f ? find_part<M, WEIGH>(p, rank, lane) : find_tile<M>(p, rank, lane);
}

// Workgroup -> (key head, rank).  Ids go round-robin over the XCDs: the heads are dealt to the XCDs, so that the
// tiles that read one head's keys share an L2.
__device__ __forceinline__ void deal_head(const ServeParams& p, int id, int& head, int& rank) {
  const int X = p.n_xcd;
  if (p.Hk % X == 0) {
    const int per = p.Hk / X, xcd = id % X, slot = id / X;
    head = xcd * per + slot % per;
    rank = slot / per;
  } else if (X % p.Hk == 0) {
    const int per = X / p.Hk, xcd = id % X;
    head = xcd % p.Hk;
    rank = id / X * per + xcd / p.Hk;
  } else {
    rank = int(divide(uint32_t(id), p.heads));
    head = id - rank * p.Hk;
  }
}

// Rows of tokens behind the last sequence are zeros: their workgroups are those from number `units` on, which have no unit.
template <int D>
__device__ void clear_rows(const ServeParams& p, int head, int rank, int units, int ranks, int tid, int threads) {
  if (rank < units) return;
  int used = p.cu[p.B];
  used = used < 0 ? 0 : used;
  for (int64_t t = int64_t(used) + (rank - units); t < p.T; t += ranks - units) {
    const int64_t row = (t * p.Hk + head) * p.G;
    for (int i = tid; i < p.G * (D / 8); i += threads) *reinterpret_cast<u32x4_t*>(p.o + row * D + i * 8) = u32x4_t{0u, 0u, 0u, 0u};
    if (p.lse != nullptr)
      for (int i = tid; i < p.G; i += threads) p.lse[row + i] = -INFINITY;
  }
}

// Keys or values of one head of one sequence: resources of the rows from `row` on that end with the sequence, so that
// rows behind it arrive as zeros whatever lies there.
struct PackedRows {
  const uint16_t* base;
  uint32_t pitch;  // bytes from row to row
  int kv;
  template <int D>
  __device__ __forceinline__ i32x4_t rows(int row) const {
    const int left = kv - row;
    const uint64_t bytes = left > 0 ? uint64_t(left - 1) * pitch + uint64_t(D * 2) : 0u;
    return make_buffer_resource(reinterpret_cast<const uint8_t*>(base) + int64_t(row) * pitch,
                                bytes > 0xffffffffu ? 0xffffffffu : uint32_t(bytes));
  }
};

// The page numbers of a sequence, 64 at a time in the lanes of a wave.
struct PageWindow {
  int32_t pages;  // of the entries 64 * at .. 64 * at + 63
  int at;
  __device__ __forceinline__ void load(const ServeParams& p, int b, int window, int lane) {
    at = window;
    const int64_t i = int64_t(window) * 64 + lane;
    int32_t page = i < p.max_pages ? p.page_table[int64_t(b) * p.max_pages + i] : 0;
    page = page < 0 ? 0 : (page >= p.num_pages ? p.num_pages - 1 : page);  // (never a fault)
    pages = page;
  }
};

// cap tanh(x / cap) of the scores.
template <int NTL>
__device__ __forceinline__ void cap_scores(f32x16_t (&st)[NTL], float cap, float c2) {
  static_for<16 * NTL>([&](auto ec) {
    constexpr int e = decltype(ec)::value;
    const float ex = __builtin_amdgcn_exp2f(st[e / 16][e % 16] * c2);
    st[e / 16][e % 16] = __builtin_fmaf(__builtin_amdgcn_rcpf(ex + 1.f), -2.f * cap, cap);
  });
}
// Scores of keys behind `limit` (the row's last key, counted from the step's first) become -inf.  Register r of tile t
// holds key 32 t + 8 (r / 4) + 4 g + r % 4.
template <int NTL>
__device__ __forceinline__ void mask_scores(f32x16_t (&st)[NTL], int limit, int g) {
  static_for<16 * NTL>([&](auto ec) {
    constexpr int e = decltype(ec)::value, t = e / 16, r = e % 16;
    constexpr int key = 32 * t + 8 * (r >> 2) + (r & 3);
    if (key + 4 * g > limit) st[t][r] = -INFINITY;
  });
}
template <int NTL>
__device__ __forceinline__ float max_of(const f32x16_t (&st)[NTL], float sl2) {
  float a = vmax(st[0][0], st[0][1]), b = vmax(st[0][2], st[0][3]);
  static_for<8 * NTL - 2>([&](auto ic) {
    constexpr int e = 2 * decltype(ic)::value + 4;
    float& m = e & 2 ? b : a;
    m = vmax3(m, st[e / 16][e % 16], st[e / 16][e % 16 + 1]);
  });
  return pair_max(vmax(a, b)) * sl2;
}

// What the joining kernel needs to know of the unit's tokens; the first part of a tile tells it.
template <int M>
__device__ __forceinline__ void tell_joins(const ServeParams& p, const Unit& u, int head, int rows_all, int tid) {
  typedef __attribute__((ext_vector_type(4))) int32_t i32x4;
  if (p.share == 0.f || head != 0 || u.step0 != 0 || tid >= M) return;
  const int row = u.tile * M + tid;
  if (row >= rows_all) return;
  const int token = int(divide(uint32_t(row), p.group));
  *reinterpret_cast<i32x4*>(p.joins + (int64_t(u.seq.first) + token) * 4) = i32x4{u.seq.first, u.parts, u.base, 0};
}

// Where a unit's results go.
template <bool BF16, int D, int M>
__device__ __forceinline__ void store_rows(const ServeParams& p, const Unit& u, int head, int slot, int row0, int rows_all,
                                           f32x16_t (&ot)[D / 32], float m_run, float l_run, uint32_t skip, uint16_t* stage,
                                           int lane) {
  // row0: first row of the wave in the sequence; slot: the part's place; skip: rows that are left out, by bit
  const int c = lane & 31, g = lane >> 5;
  const float l = pair_sum(l_run);
  if (u.part) {
    const int in_tile = (row0 & (M - 1)) + c;
    if (row0 + c < rows_all && !(skip >> c & 1)) {
      float* at = p.sums + ((int64_t(slot) * p.Hk + head) * M + in_tile) * D;
      typedef __attribute__((ext_vector_type(4))) float f32x4_t;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4)
          *reinterpret_cast<f32x4_t*>(at + 32 * dt + 8 * r4 + 4 * g) =
              f32x4_t{ot[dt][4 * r4], ot[dt][4 * r4 + 1], ot[dt][4 * r4 + 2], ot[dt][4 * r4 + 3]};
      if (g == 0) {
        float* st = p.stats + ((int64_t(slot) * p.Hk + head) * M + in_tile) * 2;
        st[0] = m_run;
        st[1] = l;
      }
    }
    return;
  }
  const bool live = l > 0.f || l != l;  // (sums that are no number stay so)
  const float inv = live ? 1.f / l : 0.f;
  // whole rows through LDS, so that a store instruction writes whole lines
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      u32x2_t ov;
      ov[0] = pack2<BF16>(ot[dt][4 * r4 + 0] * inv, ot[dt][4 * r4 + 1] * inv);
      ov[1] = pack2<BF16>(ot[dt][4 * r4 + 2] * inv, ot[dt][4 * r4 + 3] * inv);
      *reinterpret_cast<u32x2_t*>(stage + c * D + ((4 * dt + r4) ^ k_swizzle<D>(c)) * 8 + 4 * g) = ov;
    }
  constexpr int CPR = D / 8, RPS = 64 / CPR;
  // (rows of o: the wave's first token and head, and 32-bit offsets from there)
  const int pch = lane % CPR, token0 = __builtin_amdgcn_readfirstlane(int(divide(uint32_t(row0), p.group)));
  uint16_t* const o = p.o + (int64_t(u.seq.first + token0) * p.Hk + head) * p.G * D;
  const uint32_t token_step = uint32_t(p.Hk * p.G - p.G) * D;
#pragma unroll
  for (int i = 0; i < 32 / RPS; ++i) {
    const int row = i * RPS + lane / CPR;
    const u32x4_t val = *reinterpret_cast<const u32x4_t*>(stage + row * D + pch * 8);
    const int r = row0 + row;
    if (r < rows_all && !(skip >> row & 1)) {
      // (token - token0) heads of all groups and r - token G of this one: r - token0 G of this one, and the tokens' rest
      const uint32_t token = divide(uint32_t(r), p.group) - uint32_t(token0);
      const uint32_t at = token * token_step + uint32_t(r - token0 * p.G) * D + uint32_t(pch ^ k_swizzle<D>(row)) * 8u;
      *reinterpret_cast<u32x4_t*>(o + at) = val;
    }
  }
  if (p.lse != nullptr && g == 0 && row0 + c < rows_all && !(skip >> c & 1)) {
    const int token = int(divide(uint32_t(row0 + c), p.group));
    p.lse[(int64_t(u.seq.first + token) * p.Hk + head) * p.G + (row0 + c - token * p.G)] =
        live ? (m_run + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
  }
}

template <bool BF16, int D, bool PAGED>
__device__ __forceinline__ const uint16_t* key_row(const ServeParams& p, const Unit& u, int head, int key, bool is_v) {
  if constexpr (PAGED) {
    int page = p.page_table[int64_t(u.b) * p.max_pages + (key >> p.page_shift)];
    page = page < 0 ? 0 : (page >= p.num_pages ? p.num_pages - 1 : page);
    return (is_v ? p.v : p.k) + (((int64_t(page) * p.Hk + head) << p.page_shift) + (key & ((1 << p.page_shift) - 1))) * D;
  } else {
    const RowStrides& at = is_v ? p.v_at : p.k_at;
    return (is_v ? p.v : p.k) + (int64_t(u.seq.first) + key) * at.row + head * at.h;
  }
}
template <bool BF16>
__device__ __forceinline__ float widen16(uint32_t x) {
  if constexpr (BF16) {
    return __builtin_bit_cast(float, x << 16);
  } else {
    return float(__builtin_bit_cast(_Float16, uint16_t(x)));
  }
}
// A step's scores become weights, packed for the second product; the row's maximum is kept exactly, its sums follow.
template <bool BF16, int NTL, int DT>
__device__ __forceinline__ void weigh_step(const f32x16_t (&st)[NTL], float sl2, float& m_run, float& l_run, f32x16_t (&ot)[DT],
                                           u32x4_t (&pb)[NTL][2]) {
  const float m_new = fmaxf(m_run, max_of<NTL>(st, sl2));
  if (__builtin_amdgcn_ballot_w64(m_new != m_run) != 0) {
    const float m_old = m_run == -INFINITY ? (m_new == -INFINITY ? 0.f : m_new) : m_run;
    const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_old - m_new);
    l_run *= alpha;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) ot[dt][r] *= alpha;
    m_run = m_new;
  }
  const float m_ref = m_run == -INFINITY ? 0.f : m_run;
  static_for<8 * NTL>([&](auto ic) {
    constexpr int i = decltype(ic)::value, t = i / 8, r = 2 * (i % 8);
    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[t][r], sl2, -m_ref));
    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[t][r + 1], sl2, -m_ref));
    l_run += p0 + p1;
    pb[t][r >> 3][(r & 7) >> 1] = pack2<BF16>(p0, p1);
  });
}

// Rows whose sums are no numbers, in a unit where rows attend different keys: a weight of zero times a value that is
// infinite or no number, of a key that the row does not attend, may have made them so.  Such rows of a wave (and those that
// are no numbers by right) are summed again.  Up to the key that the wave's first row attends last nothing is masked, and
// matrix products do it, from memory without LDS; of the keys behind, as many as the wave has tokens at most, a row adds one at a
// time those that it attends.  Packed prompts with a value that is no number in the first key, which spoils every row, or in
// the last, which spoils one: 4096 tokens, 8 / 2 heads, D=128, 0.70 ms, 0.07 without one; 8192 tokens, 8 heads 2.1 and 0.17;
// 512 tokens, 8 heads, D=64 0.07 and 0.01 (a row at a time over all of its keys, a lane per key: 21, 47 and 2.2 ms).
template <bool BF16, int D, int M, bool PAGED>
__device__ __forceinline__ void sum_rows_again(const ServeParams& p, const Unit& u, int head, int slot, int row0, uint32_t rows, int from,
                               int to, int lane) {
  typedef __attribute__((ext_vector_type(4))) float f32x4_t;
  constexpr int KS = D / 16, DT = D / 32, STEP = 32;
  const int g = lane >> 5, c = lane & 31, shift = u.seq.kv - u.seq.n, rows_all = u.seq.n * p.G;
  const int row = row0 + c < rows_all ? row0 + c : rows_all - 1, token = int(divide(uint32_t(row), p.group));
  const int last_row = row0 + 32 < rows_all ? row0 + 31 : rows_all - 1;
  const int limit = shift + token;  // the row's last key
  const int first_key = __builtin_amdgcn_readfirstlane(shift + int(divide(uint32_t(row0), p.group)));
  const int last_key = __builtin_amdgcn_readfirstlane(shift + int(divide(uint32_t(last_row), p.group)));
  const int common = first_key + 1 < to ? first_key + 1 : to, end = last_key + 1 < to ? last_key + 1 : to;
  u32x4_t qf[KS];
  {
    const uint16_t* at = p.q + int64_t(u.seq.first + token) * p.q_row + int64_t(head * p.G + (row - token * p.G)) * p.q_head;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const u32x4_t*>(at + 16 * s + 8 * g);
  }
  f32x16_t ot[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) ot[dt] = f32x16_t{};
  float m_run = -INFINITY, l_run = 0.f;
  for (int key0 = from; key0 < common; key0 += STEP) {
    const int key = key0 + c < common ? key0 + c : common - 1;
    const uint16_t* k = key_row<BF16, D, PAGED>(p, u, head, key, false);
    const int64_t v = key_row<BF16, D, PAGED>(p, u, head, key, true) - p.v;
    f32x16_t st[1];
    st[0] = f32x16_t{};
#pragma unroll
    for (int s = 0; s < KS; ++s) st[0] = mfma_32x32x16<BF16>(*reinterpret_cast<const u32x4_t*>(k + 16 * s + 8 * g), qf[s], st[0]);
    if (p.softcap > 0.f) cap_scores<1>(st, p.softcap, p.cap_c2);
    if (key0 + STEP > common) mask_scores<1>(st, common - 1 - key0, g);
    u32x4_t pb[1][2];
    weigh_step<BF16, 1>(st, p.sl2, m_run, l_run, ot, pb);
#pragma unroll
    for (int ts = 0; ts < 2; ++ts) {
      // the keys 16 ts + 4 g + (0 .. 3) and 8 further on, a dimension per lane
      int64_t at[8];
      bool in[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int n = 16 * ts + 4 * g + (i & 3) + 8 * (i >> 2);
        at[i] = __shfl(v, n) + c;
        in[i] = key0 + n < common;
      }
      static_for<DT>([&](auto dc) {
        constexpr int dt = decltype(dc)::value;
        uint32_t x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = in[i] ? p.v[at[i] + 32 * dt] : 0u;
        ot[dt] = mfma_32x32x16<BF16>(u32x4_t{x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16}, pb[0][ts], ot[dt]);
        __builtin_amdgcn_sched_barrier(0);
      });
    }
  }
  for (int key = common < from ? from : common; key < end; ++key) {
    const uint16_t* k = key_row<BF16, D, PAGED>(p, u, head, key, false);
    const uint16_t* v = key_row<BF16, D, PAGED>(p, u, head, key, true);
    float x = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const u32x4_t y = *reinterpret_cast<const u32x4_t*>(k + 16 * s + 8 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x = __builtin_fmaf(widen16<BF16>(qf[s][i] & 0xffffu), widen16<BF16>(y[i] & 0xffffu), x);
        x = __builtin_fmaf(widen16<BF16>(qf[s][i] >> 16), widen16<BF16>(y[i] >> 16), x);
      }
    }
    x = pair_sum(x);
    if (p.softcap > 0.f)
      x = __builtin_fmaf(__builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * p.cap_c2) + 1.f), -2.f * p.softcap, p.softcap);
    x *= p.sl2;
    if (key > limit) continue;
    const float m_new = fmaxf(m_run, x), m_ref = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_ref), weight = __builtin_amdgcn_exp2f(x - m_ref);
    l_run = __builtin_fmaf(l_run, alpha, g == 0 ? weight : 0.f);
    m_run = m_new;
    static_for<4 * DT>([&](auto ic) {
      constexpr int dt = decltype(ic)::value / 4, r = 4 * (decltype(ic)::value % 4);
      const u32x2_t y = *reinterpret_cast<const u32x2_t*>(v + 32 * dt + 2 * r + 4 * g);
      const float f[4] = {widen16<BF16>(y[0] & 0xffffu), widen16<BF16>(y[0] >> 16), widen16<BF16>(y[1] & 0xffffu), widen16<BF16>(y[1] >> 16)};
#pragma unroll
      for (int i = 0; i < 4; ++i) ot[dt][r + i] = __builtin_fmaf(weight, f[i], ot[dt][r + i] * alpha);
    });
  }
  const float l = pair_sum(l_run);
  if (!(rows >> c & 1)) return;
  const bool live = l > 0.f || l != l;
  const float inv = live ? 1.f / l : 0.f;
  const int64_t at = (int64_t(u.seq.first + token) * p.Hk + head) * p.G + (row - token * p.G);
  const int64_t part_at = (int64_t(slot) * p.Hk + head) * M + (row & (M - 1));
  static_for<4 * DT>([&](auto ic) {
    constexpr int dt = decltype(ic)::value / 4, r = 4 * (decltype(ic)::value % 4);
    const int d = 32 * dt + 2 * r + 4 * g;
    if (u.part) {
      *reinterpret_cast<f32x4_t*>(p.sums + part_at * D + d) = f32x4_t{ot[dt][r], ot[dt][r + 1], ot[dt][r + 2], ot[dt][r + 3]};
    } else {
      const u32x2_t ov = {live ? pack2<BF16>(ot[dt][r] * inv, ot[dt][r + 1] * inv) : 0u, live ? pack2<BF16>(ot[dt][r + 2] * inv, ot[dt][r + 3] * inv) : 0u};
      *reinterpret_cast<u32x2_t*>(p.o + at * D + d) = ov;
    }
  });
  if (g != 0) return;
  if (u.part) {
    p.stats[part_at * 2] = m_run;
    p.stats[part_at * 2 + 1] = l;
  } else if (p.lse != nullptr) {
    p.lse[at] = live ? (m_run + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
  }
}
// The rows of a wave whose O holds something that is no number (or infinite), bit by row.
template <int DT>
__device__ __forceinline__ uint32_t odd_rows(const f32x16_t (&ot)[DT]) {
  float x = 0.f;
  static_for<16 * DT>([&](auto ec) {
    constexpr int e = decltype(ec)::value;
    x = __builtin_fmaf(ot[e / 16][e % 16], 0.f, x);
  });
  const uint64_t odd = __builtin_amdgcn_ballot_w64(!(x == 0.f));
  return uint32_t(odd) | uint32_t(odd >> 32);
}

__device__ __forceinline__ uint32_t live_rows(int rows) { return rows >= 32 ? ~0u : (rows <= 0 ? 0u : (1u << rows) - 1u); }

// KG groups of waves have shared the steps of a tile: every wave's maxima and sums, and its O, go into its own place in LDS
// (wave_at of its group's bytes, which nobody reads any more); then each group adds up and stores a share of the columns
// against the common maximum.
template <int D>
constexpr size_t kMergeBytes = size_t(32) * D * 4 + 256;  // of a wave
template <bool BF16, int D, int M, int KG, bool PAGED>
__device__ __forceinline__ void merge_groups(const ServeParams& p, const Unit& u, int head, int slot, int row0, int rows_all,
                                             const f32x16_t (&ot)[D / 32], float m_run, float l_run, bool several,
                                             uint8_t* lds, size_t group_bytes, size_t wave_at, int kg, int from, int to, int lane) {
  typedef __attribute__((ext_vector_type(4))) float f32x4_t;
  constexpr int PIECES = D / 8, MINE = PIECES / KG;  // 4-register pieces of a lane's O
  static_assert(PIECES % KG == 0, "every group has a share");
  const int c = lane & 31, g = lane >> 5;
  auto piece_at = [&](int i, int piece) { return reinterpret_cast<f32x4_t*>(lds + i * group_bytes + wave_at) + piece * 64 + lane; };
  auto stat_at = [&](int i) { return reinterpret_cast<float*>(lds + i * group_bytes + wave_at + 32 * D * 4) + 2 * c; };
  const float l = pair_sum(l_run);
  const uint32_t mine_odd = several ? odd_rows<D / 32>(ot) : 0u;
  if (g == 0) {
    stat_at(kg)[0] = m_run;
    stat_at(kg)[1] = mine_odd >> c & 1 ? __builtin_nanf("") : l;
  }
  static_for<PIECES>([&](auto pc) {
    constexpr int piece = decltype(pc)::value, dt = piece / 4, r = 4 * (piece % 4);
    *piece_at(kg, piece) = f32x4_t{ot[dt][r], ot[dt][r + 1], ot[dt][r + 2], ot[dt][r + 3]};
  });
  __syncthreads();
  float m_all = -INFINITY, l_all = 0.f, scale[KG];
#pragma unroll
  for (int i = 0; i < KG; ++i) m_all = fmaxf(m_all, stat_at(i)[0]);
  const float m_ref = m_all == -INFINITY ? 0.f : m_all;
#pragma unroll
  for (int i = 0; i < KG; ++i) {
    scale[i] = __builtin_amdgcn_exp2f(stat_at(i)[0] - m_ref);
    l_all += stat_at(i)[1] * scale[i];
  }
  const bool live = l_all > 0.f || l_all != l_all;
  const float inv = u.part ? 1.f : (live ? 1.f / l_all : 0.f);
  const uint32_t odd = several ? uint32_t(__builtin_amdgcn_ballot_w64(l_all != l_all)) & live_rows(rows_all - row0) : 0u;
  const bool mine = row0 + c < rows_all && !(odd >> c & 1);
  const int row = row0 + c < rows_all ? row0 + c : rows_all - 1, token = int(divide(uint32_t(row), p.group));
  const int64_t at = (int64_t(u.seq.first + token) * p.Hk + head) * p.G + (row - token * p.G);
  const int64_t part_at = (int64_t(slot) * p.Hk + head) * M + (row0 & (M - 1)) + c;
#pragma unroll
  for (int n = 0; n < MINE; ++n) {
    const int piece = kg * MINE + n;
    f32x4_t x = *piece_at(0, piece) * scale[0];
#pragma unroll
    for (int i = 1; i < KG; ++i) x += *piece_at(i, piece) * scale[i];
    if (!mine) continue;
    if (u.part) {
      *reinterpret_cast<f32x4_t*>(p.sums + part_at * D + 8 * piece + 4 * g) = x;
    } else {
      const u32x2_t ov = {live ? pack2<BF16>(x[0] * inv, x[1] * inv) : 0u, live ? pack2<BF16>(x[2] * inv, x[3] * inv) : 0u};
      *reinterpret_cast<u32x2_t*>(p.o + at * D + 8 * piece + 4 * g) = ov;
    }
  }
  if (kg == 0 && g == 0 && mine) {
    if (u.part) {
      p.stats[part_at * 2] = m_all;
      p.stats[part_at * 2 + 1] = l_all;
    } else if (p.lse != nullptr) {
      p.lse[at] = live ? (m_all + __builtin_amdgcn_logf(l_all)) * 0.6931471805599453f : -INFINITY;
    }
  }
  if (kg == 0 && odd != 0) sum_rows_again<BF16, D, M, PAGED>(p, u, head, slot, row0, odd, from, to, lane);
}

// Rows from `row` on of the page that a step reads, up to `to`.
template <int D>
__device__ __forceinline__ i32x4_t page_rows(const ServeParams& p, const uint16_t* pages, const PageWindow& win, int head, int row, int to) {
  const int page = __builtin_amdgcn_readlane(win.pages, (row >> p.page_shift) & 63);
  const int64_t at = (((int64_t(page) * p.Hk + head) << p.page_shift) + (row & ((1 << p.page_shift) - 1))) * D;
  int left = to - row;
  left = left < 0 ? 0 : (left > kPageOfStep ? kPageOfStep : left);
  return make_buffer_resource(pages + at, uint32_t(left) * (D * 2u));
}

// ---- few rows ---------------------------------------------------------------------------------------------------
//
// Single tokens, a few, and short prompts: tiles of 32 rows.  The work is the reading of K and V: a wave has a K and a V
// tile of its own in LDS; the loads of the next K go out once the scores have been made of this one, those of the next V
// behind the second product, and nothing waits for another wave.  KG waves of a workgroup share the steps of a unit (wave
// i takes the steps i, i + KG, ...) and add up their results in LDS.

template <int D>
constexpr int kFewStep = D == 128 ? 32 : 64;  // keys per step: 16 KiB of K and V
template <int D>
constexpr size_t kFewLdsBytes = kMergeBytes<D> > size_t(2) * kFewStep<D> * D * 2 ? kMergeBytes<D> : size_t(2) * kFewStep<D> * D * 2;  // of a wave

// The rows from row0 on of a unit, by one wave, or by KG of which this is number kg.  LDS: bytes of a wave from lds on.
template <bool BF16, int D, Keys KEYS, int M, int KG, int STEP, size_t LDS>
__device__ __forceinline__ void few_rows(const ServeParams& p, const Unit& u, int head, int slot, int row0, int kg, uint8_t* lds, int lane) {
  constexpr bool PAGED = KEYS != kPacked;
  constexpr int NTL = STEP / 32, KS = D / 16, DT = D / 32, CPR = D / 8;
  constexpr int RPC = 64 / CPR, NCH = STEP / RPC, TILE = STEP * D;  // rows per load, loads per tile
  constexpr int KPER = RPC % 16 == 0 ? 1 : 16 / RPC;
  static_assert(LDS >= size_t(2) * TILE * 2, "a tile of K and one of V");
  uint16_t* sK = reinterpret_cast<uint16_t*>(lds + kg * LDS);
  uint16_t* sV = sK + TILE;
  const int g = lane >> 5, c = lane & 31;
  const int rows_all = u.seq.n * p.G;
  const int row = row0 + c < rows_all ? row0 + c : rows_all - 1;
  const int token = int(divide(uint32_t(row), p.group));
  const int limit = p.causal ? u.seq.kv - u.seq.n + token : u.seq.kv - 1;  // the row's last key
  const int last_row = row0 + 32 < rows_all ? row0 + 31 : rows_all - 1;
  const int last_key = p.causal ? u.seq.kv - u.seq.n + int(divide(uint32_t(last_row), p.group)) : u.seq.kv - 1;
  const int first_key = p.causal ? u.seq.kv - u.seq.n + int(divide(uint32_t(row0), p.group)) : u.seq.kv - 1;
  const int from = u.step0 * kStepKeys;
  int to = u.steps < steps_of(u.seq.kv) - u.step0 ? (u.step0 + u.steps) * kStepKeys : u.seq.kv;
  if (to > last_key + 1) to = last_key + 1;  // (keys at or behind `to` are not read)
  const int nsteps = to > from ? (to - from + STEP - 1) / STEP : 0;

  u32x4_t qf[KS];
  {
    const uint16_t* at = p.q + int64_t(u.seq.first + token) * p.q_row + int64_t(head * p.G + (row - token * p.G)) * p.q_head;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const u32x4_t*>(at + 16 * s + 8 * g);
  }

  // Direct loads: instruction i of a tile fills the rows i * RPC .. i * RPC + RPC - 1.
  const int ld_row = lane / CPR, ld_pch = lane % CPR;
  PackedRows kr, vr;
  PageWindow window{0, -1};
  uint32_t kpitch = D * 2, vpitch = D * 2;
  if constexpr (!PAGED) {
    kr = {p.k + int64_t(u.seq.first) * p.k_at.row + head * p.k_at.h, p.k_at.row * 2u, to};
    vr = {p.v + int64_t(u.seq.first) * p.v_at.row + head * p.v_at.h, p.v_at.row * 2u, to};
    kpitch = kr.pitch;
    vpitch = vr.pitch;
  }
  uint32_t koff[KPER];
#pragma unroll
  for (int i = 0; i < KPER; ++i) koff[i] = uint32_t(ld_row) * kpitch + uint32_t(ld_pch ^ k_swizzle<D>(ld_row + i * RPC)) * 16u;
  const uint32_t voff = uint32_t(ld_row) * vpitch + uint32_t((((ld_pch >> 1) ^ v_swizzle<D>(ld_row)) << 1) | (ld_pch & 1)) * 16u;
  const uint32_t lds_k = lds_offset_of(sK), lds_v = lds_offset_of(sV);
  auto need_window = [&](int key0) {
    if constexpr (PAGED) {
      const int n = (key0 >> p.page_shift) >> 6;
      if (n != window.at) window.load(p, u.b, n, lane);
    }
  };
  auto issue = [&](bool is_v, int key0) {
    i32x4_t r;
    if constexpr (KEYS == kPacked) r = is_v ? vr.rows<D>(key0) : kr.rows<D>(key0);
    if constexpr (KEYS == kPages) r = page_rows<D>(p, is_v ? p.v : p.k, window, head, key0, to);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const uint32_t dst = (is_v ? lds_v : lds_k) + uint32_t(i) * 1024u, off = is_v ? voff : koff[i % KPER];
      if constexpr (KEYS == kSmallPages) {
        const int key = key0 + i * RPC;
        const int page = __builtin_amdgcn_readlane(window.pages, (key >> p.page_shift) & 63);
        const int64_t at = (((int64_t(page) * p.Hk + head) << p.page_shift) + (key & ((1 << p.page_shift) - 1))) * D;
        int left = to - key;
        left = left < 0 ? 0 : (left > RPC ? RPC : left);
        buffer_to_lds_b128(make_buffer_resource((is_v ? p.v : p.k) + at, uint32_t(left) * (D * 2u)), off, 0, dst);
      } else {
        buffer_to_lds_b128(r, off, uint32_t(i * RPC) * (is_v ? vpitch : kpitch), dst);
      }
    }
  };

  const f32x16_t zero16 = {};
  f32x16_t ot[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) ot[dt] = zero16;
  float m_run = -INFINITY, l_run = 0.f;
  const int i16 = c & 15, j16 = c >> 4;
  if (kg < nsteps) {
    need_window(from + kg * STEP);
    issue(false, from + kg * STEP);
    issue(true, from + kg * STEP);
  }
  const uint16_t* tK = sK;
  const uint16_t* tV = sV;
  for (int it = kg; it < nsteps; it += KG) {
    const int key0 = from + it * STEP;
    const bool more = it + KG < nsteps;
    wait_loads_but<NCH>();  // V may be under way
    f32x16_t st[NTL];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int t = 0; t < NTL; ++t) {
        const int r = 32 * t + c;
        const u32x4_t a = *reinterpret_cast<const u32x4_t*>(tK + r * D + ((2 * s + g) ^ k_swizzle<D>(r)) * 8);
        st[t] = mfma_32x32x16<BF16>(a, qf[s], s == 0 ? zero16 : st[t]);
      }
    if (more) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K has been read
      need_window(key0 + KG * STEP);
      issue(false, key0 + KG * STEP);
    }
    if (p.softcap > 0.f) cap_scores<NTL>(st, p.softcap, p.cap_c2);
    if (key0 + STEP - 1 > first_key || key0 + STEP > to) {
      const int stop = limit < to - 1 ? limit : to - 1;
      mask_scores<NTL>(st, stop - key0, g);
    }
    u32x4_t pb[NTL][2];
    weigh_step<BF16, NTL>(st, p.sl2, m_run, l_run, ot, pb);
    if (more) {
      wait_loads_but<NCH>();  // the next K may be under way
    } else {
      wait_loads();
    }
#pragma unroll
    for (int j = 0; j < (STEP / 16) * DT; ++j) {
      const int ts = j / DT, dt = j % DT;
      const int vrow = 16 * ts + 4 * g + (i16 >> 2), unit = 2 * dt + j16;
      const s16x4_t lo = lds_read_tr16(tV + vrow * D + (unit ^ v_swizzle<D>(vrow)) * 16 + (i16 & 3) * 4);
      const s16x4_t hi = lds_read_tr16(tV + (vrow + 8) * D + (unit ^ v_swizzle<D>(vrow + 8)) * 16 + (i16 & 3) * 4);
      const u32x2_t lo2 = __builtin_bit_cast(u32x2_t, lo), hi2 = __builtin_bit_cast(u32x2_t, hi);
      ot[dt] = mfma_32x32x16<BF16>(u32x4_t{lo2[0], lo2[1], hi2[0], hi2[1]}, pb[ts >> 1][ts & 1], ot[dt]);
    }
    if (more) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V has been read
      issue(true, key0 + KG * STEP);
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  const bool several = p.causal && first_key < last_key;  // rows that attend different keys
  if constexpr (KG == 1) {
    const uint32_t odd = several ? odd_rows<DT>(ot) & live_rows(rows_all - row0) : 0u;
    store_rows<BF16, D, M>(p, u, head, slot, row0, rows_all, ot, m_run, l_run, odd, sK, lane);
    if (odd != 0) sum_rows_again<BF16, D, M, PAGED>(p, u, head, slot, row0, odd, from, to, lane);
  } else {
    merge_groups<BF16, D, M, KG, PAGED>(p, u, head, slot, row0, rows_all, ot, m_run, l_run, several, lds,
                                        LDS, 0, kg, from, to, lane);
  }
}

template <bool BF16, int D, Keys KEYS, int KG>
__global__ void __launch_bounds__(64 * KG, 2) serve_few_kernel(const ServeParams p) {
  constexpr int M = 32;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
  const int kg = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int head, rank;
  deal_head(p, blockIdx.x, head, rank);
  if (rank >= p.units) return;
  const Unit u = find_unit<M, (KEYS != kPacked && KG == 4)>(p, rank, lane);
  if (!u.found) {  // (with parts the joining kernel clears rows behind the last sequence)
    if (p.share == 0.f) clear_rows<D>(p, head, rank, u.step0, p.units, threadIdx.x, 64 * KG);
    return;
  }
  tell_joins<M>(p, u, head, u.seq.n * p.G, threadIdx.x);
  few_rows<BF16, D, KEYS, M, KG, kFewStep<D>, kFewLdsBytes<D>>(p, u, head, u.slot, u.tile * M, kg, lds_raw, lane);
}

// ---- many rows: four waves per unit -------------------------------------------------------------------------------
//
// A tile of M rows, 32 per wave, walks its keys in steps, software-pipelined like the block-sparse forward: iteration i issues the matrix instructions of S^T(i + 1) and of O^T += V^T P^T(i - 1) in slots, and between
// them the softmax of step i, the operand fetches and the loads of K(i + 2) and V(i).  The exponentials' reference
// stays where it is as long as the row sums do not outgrow it.
// M = 128: four waves, steps of 64 keys.  M = 64: two groups of two waves share the steps (group i takes the steps i, i + 2,
// ...) and add up at the end: half the walk, for launches that a few tiles' walks are long for; steps of 32 keys at
// head_dim 128, so that two workgroups share a compute unit there too.

template <int D, int M>
constexpr int kTileStep = M == 64 && D == 128 ? 32 : 64;
// Of a group: two sets of K and V, or its waves' sums.
template <int D, int M>
constexpr size_t kTileLdsBytes = M == 64 && 2 * kMergeBytes<D> > size_t(8) * kTileStep<D, M> * D ? 2 * kMergeBytes<D>
                                                                                             : size_t(8) * kTileStep<D, M> * D;

// Sequences of so few keys gain nothing from a pipeline over their steps: each wave has its rows' walk to itself and waits for
// nobody.  32 / 8 heads, D=128: 4096 prompts of 20 - 40 tokens 642 us, 729 in the pipeline; 300 of 40 - 80 tokens 95 and 102;
// 1000 of 67 - 133 tokens 540 and 545; 1000 of 15 and one of 4000 223 and 246 (300 of 133 - 267, beyond the line, D=64, 16
// heads 190 and 184).
constexpr int kShortKeys = 128;

template <bool BF16, int D, Keys KEYS, int M>
__global__ void __launch_bounds__(256, 2) serve_tile_kernel(const ServeParams p) {
  constexpr bool PAGED = KEYS != kPacked;
  constexpr int KG = 128 / M, W = M / 32, STEP = kTileStep<D, M>, NTL = STEP / 32, KS = D / 16, DT = D / 32, CPR = D / 8;
  constexpr int TILE = STEP * D;
  constexpr int RPC = 64 / CPR;            // rows filled by a wave's load
  constexpr int ROW_STRIDE = RPC * W;      // rows between a thread's loads
  constexpr int NCH = STEP / ROW_STRIDE;   // loads per thread and tile
  constexpr int KPER = ROW_STRIDE % 16 == 0 ? 1 : 16 / ROW_STRIDE;
  static_assert((KPER * ROW_STRIDE) % 16 == 0 && ROW_STRIDE % 4 == 0 && RPC <= 16, "swizzles repeat over a thread's loads");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
  const int tid = threadIdx.x & (64 * W - 1), lane = tid & 63, g = lane >> 5, c = lane & 31;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kg = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(int(threadIdx.x) / (64 * W));
  uint16_t* sK = reinterpret_cast<uint16_t*>(lds_raw + kg * kTileLdsBytes<D, M>);  // [2][TILE]
  uint16_t* sV = sK + 2 * TILE;
  int head, rank;
  deal_head(p, blockIdx.x, head, rank);
  if (rank >= p.units) return;
  const Unit u = find_unit<M, M == 128 && PAGED>(p, rank, lane);
  if (!u.found) {
    if (p.share == 0.f) clear_rows<D>(p, head, rank, u.step0, p.units, threadIdx.x, 256);
    return;
  }
  if constexpr (M == 128) {
    if (p.share == 0.f && u.seq.kv <= kShortKeys) {
      constexpr size_t kOwn = kTileLdsBytes<D, M> / 4;
      const int row0 = u.tile * M + 32 * w;
      if (row0 < u.seq.n * p.G) few_rows<BF16, D, KEYS, M, 1, 32, kOwn>(p, u, head, u.slot, row0, 0, lds_raw + w * kOwn, lane);
      return;
    }
  }
  const int shift = u.seq.kv - u.seq.n;  // a token's position, less its number
  const int rows_all = u.seq.n * p.G, row0 = u.tile * M + 32 * w;
  tell_joins<M>(p, u, head, rows_all, threadIdx.x);
  const int row = row0 + c < rows_all ? row0 + c : rows_all - 1;
  const int token = int(divide(uint32_t(row), p.group));
  const int last_row = u.tile * M + M < rows_all ? u.tile * M + M - 1 : rows_all - 1;
  const int last_key = p.causal ? shift + int(divide(uint32_t(last_row), p.group)) : u.seq.kv - 1;
  const int wave_first = row0 < rows_all ? row0 : rows_all - 1;
  const int first_key = __builtin_amdgcn_readfirstlane(p.causal ? shift + int(divide(uint32_t(wave_first), p.group)) : u.seq.kv - 1);
  const int from = u.step0 * kStepKeys;
  int to = u.steps < steps_of(u.seq.kv) - u.step0 ? (u.step0 + u.steps) * kStepKeys : u.seq.kv;
  if (to > last_key + 1) to = last_key + 1;  // (keys at or behind `to` are not read)
  to = __builtin_amdgcn_readfirstlane(to);
  // (of each group; where one has a step less than the other its last one lies behind `to`: nothing of it is read, and all
  // its scores are masked)
  const int nsteps = __builtin_amdgcn_readfirstlane(to > from ? (to - from + STEP * KG - 1) / (STEP * KG) : 0);
  constexpr int NEXT = STEP * KG;  // keys from a group's step to its next
  const int from_kg = from + kg * STEP;

  u32x4_t qf[KS];
  {
    const uint16_t* at = p.q + int64_t(u.seq.first + token) * p.q_row + int64_t(head * p.G + (row - token * p.G)) * p.q_head;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const u32x4_t*>(at + 16 * s + 8 * g);
  }

  const int ld_row = KEYS == kSmallPages ? lane / CPR : tid / CPR, ld_pch = tid % CPR, sw_row = tid / CPR;
  PackedRows kr, vr;
  PageWindow kwin{0, -1}, vwin{0, -1};
  uint32_t kpitch = D * 2, vpitch = D * 2;
  if constexpr (!PAGED) {
    kr = {p.k + int64_t(u.seq.first) * p.k_at.row + head * p.k_at.h, p.k_at.row * 2u, to};
    vr = {p.v + int64_t(u.seq.first) * p.v_at.row + head * p.v_at.h, p.v_at.row * 2u, to};
    kpitch = kr.pitch;
    vpitch = vr.pitch;
  }
  uint32_t koff[KPER];
#pragma unroll
  for (int i = 0; i < KPER; ++i)
    koff[i] = uint32_t(ld_row) * kpitch + uint32_t(ld_pch ^ k_swizzle<D>(sw_row + i * ROW_STRIDE)) * 16u;
  const uint32_t voff = uint32_t(ld_row) * vpitch + uint32_t((((ld_pch >> 1) ^ v_swizzle<D>(sw_row)) << 1) | (ld_pch & 1)) * 16u;
  const uint32_t lds_k0 = lds_offset_of(sK) + uint32_t(w) * 1024u, lds_v0 = lds_offset_of(sV) + uint32_t(w) * 1024u;
  // Before the loads of a step's K, or V: its window of page numbers.
  auto need_window = [&](PageWindow& win, const PageWindow& other, int key0) {
    if constexpr (PAGED) {
      const int n = (key0 >> p.page_shift) >> 6;
      if (n != win.at) {
        if (n == other.at) {
          win = other;
        } else {
          win.load(p, u.b, n, lane);
        }
      }
    }
  };
  // Load n of a tile pair: n < NCH part n of V, else of K.  rk, rv: (but for small pages) the rows from the step's first on.
  auto issue_load = [&](int n, int buf, int k_key0, int v_key0, const i32x4_t& rk, const i32x4_t& rv) {
    const bool is_v = n < NCH;
    const int i = is_v ? n : n - NCH;
    const uint32_t dst = (is_v ? lds_v0 : lds_k0) + uint32_t(buf) * (TILE * 2u) + uint32_t(i) * (W * 1024u);
    const uint32_t off = is_v ? voff : koff[i % KPER];
    if constexpr (KEYS == kSmallPages) {
      const int key = (is_v ? v_key0 : k_key0) + i * ROW_STRIDE + w * RPC;
      const int page = __builtin_amdgcn_readlane(is_v ? vwin.pages : kwin.pages, (key >> p.page_shift) & 63);
      const int64_t at = (((int64_t(page) * p.Hk + head) << p.page_shift) + (key & ((1 << p.page_shift) - 1))) * D;
      int left = to - key;
      left = left < 0 ? 0 : (left > RPC ? RPC : left);
      buffer_to_lds_b128(make_buffer_resource((is_v ? p.v : p.k) + at, uint32_t(left) * (D * 2u)), off, 0, dst);
    } else {
      buffer_to_lds_b128(is_v ? rv : rk, off, uint32_t(i * ROW_STRIDE) * (is_v ? vpitch : kpitch), dst);
    }
  };
  auto rows_of = [&](bool is_v, int key0) {
    if constexpr (KEYS == kPacked) {
      return (is_v ? vr : kr).template rows<D>(key0);
    } else if constexpr (KEYS == kPages) {
      return page_rows<D>(p, is_v ? p.v : p.k, is_v ? vwin : kwin, head, key0, to);
    } else {
      return i32x4_t{};
    }
  };

  auto k_frag = [&](const uint16_t* tK, int s, int t) {
    const int r = 32 * t + c;
    return *reinterpret_cast<const u32x4_t*>(tK + r * D + ((2 * s + g) ^ k_swizzle<D>(r)) * 8);
  };
  const int i16 = c & 15, j16 = c >> 4;
  auto v_frag = [&](const uint16_t* tV, int j) {
    const int ts = j / DT, dt = j % DT;
    const int vrow = 16 * ts + 4 * g + (i16 >> 2), unit = 2 * dt + j16;
    const s16x4_t lo = lds_read_tr16(tV + vrow * D + (unit ^ v_swizzle<D>(vrow)) * 16 + (i16 & 3) * 4);
    const s16x4_t hi = lds_read_tr16(tV + (vrow + 8) * D + (unit ^ v_swizzle<D>(vrow + 8)) * 16 + (i16 & 3) * 4);
    const u32x2_t lo2 = __builtin_bit_cast(u32x2_t, lo), hi2 = __builtin_bit_cast(u32x2_t, hi);
    return u32x4_t{lo2[0], lo2[1], hi2[0], hi2[1]};
  };

  const f32x16_t zero16 = {};
  f32x16_t ot[DT];
  f32x16_t st[2][NTL];   // (written by the first products, and the first softmax)
  u32x4_t pb[2][NTL][2];
  float m_run = -INFINITY, m_ref = 0.f, l_run = 0.f, alpha_pending = 1.f;
  constexpr uint32_t kOwesRescale = 1, kOwesLook = 2;
  uint32_t owed = kOwesLook;
  constexpr int NQK = NTL * KS, NPV_ALL = (STEP / 16) * DT, NL = 2 * NCH, PF = 3;
  // (as in the block-sparse forward: how far a row may outgrow its reference before the next look, and before the
  // step itself is done again)
  constexpr float kSlack = 6.f, kGrown = 0x1p10f, kRedo = 0x1p13f;

  auto weights = [&](auto set_c, auto ic, float& s0, float& s1) {
    constexpr int SET = decltype(set_c)::value, i = decltype(ic)::value, t = i / 8, r = 2 * (i % 8);
    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[SET][t][r], p.sl2, -m_ref));
    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(st[SET][t][r + 1], p.sl2, -m_ref));
    if constexpr (i == 0) {
      s0 = p0;
      s1 = p1;
    } else {
      s0 += p0;
      s1 += p1;
    }
    uint32_t packed = pack2<BF16>(p0, p1);
    pin(packed);
    pb[SET][t][r >> 3][(r & 7) >> 1] = packed;
    pin(s0, s1);
  };
  auto set_reference = [&](float m_new) {
    m_ref = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_ref);
    l_run *= alpha;
    m_run = m_new;
    return alpha;
  };
  auto look_again = [&]() { return __builtin_amdgcn_ballot_w64(m_run == -INFINITY) != 0 ? kOwesLook : 0u; };
  auto look = [&](auto set_c) {
    constexpr int SET = decltype(set_c)::value;
    const float m_cand = max_of<NTL>(st[SET], p.sl2);
    owed = 0;
    if (__builtin_amdgcn_ballot_w64(m_cand > m_run + kSlack) != 0) {
      alpha_pending = set_reference(vmax(m_run, m_cand));
      owed = kOwesRescale;
    }
    owed |= look_again();
  };
  auto redo = [&](auto set_c, float& sum) {
    constexpr int SET = decltype(set_c)::value;
    const float alpha = set_reference(vmax(m_run, max_of<NTL>(st[SET], p.sl2)));
    alpha_pending = owed & kOwesRescale ? alpha_pending * alpha : alpha;
    float s0, s1;
    static_for<8 * NTL>([&](auto ic) { weights(set_c, ic, s0, s1); });
    sum = s0 + s1;
    owed = kOwesRescale | look_again();
  };
  auto rescale = [&]() {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) ot[dt][r] *= alpha_pending;
    owed &= ~kOwesRescale;
  };

  auto body_prefetch = [&](auto set_c, auto first_c, u32x4_t* opq) {
    constexpr int SET = decltype(set_c)::value, NPV = decltype(first_c)::value != 0 ? 0 : NPV_ALL;
    const uint16_t* tK = sK + (SET ^ 1) * TILE;
    const uint16_t* tV = sV + (SET ^ 1) * TILE;
    static_for<PF>([&](auto nc) {
      constexpr int n = decltype(nc)::value;
      opq[n] = n < NPV ? v_frag(tV, n) : k_frag(tK, (n - NPV) / NTL, (n - NPV) % NTL);
    });
  };
  auto body = [&](auto set_c, auto first_c, int k_key0, int v_key0, u32x4_t* opq) {
    constexpr int SET = decltype(set_c)::value, NPV = decltype(first_c)::value != 0 ? 0 : NPV_ALL;
    constexpr int NS = NQK + NPV;
    constexpr int LSP = (NS / 2) / NL > 0 ? (NS / 2) / NL : 1;
    constexpr int LPS = (NL * LSP + NS - 1) / NS;
    constexpr int NPR = 8 * NTL;
    const uint16_t* tK = sK + (SET ^ 1) * TILE;
    const uint16_t* tV = sV + (SET ^ 1) * TILE;
    const i32x4_t rk = rows_of(false, k_key0), rv = rows_of(true, v_key0);
    float rs0, rs1;
    __builtin_amdgcn_s_setprio(1);
    static_for<NS>([&](auto jc) {
      constexpr int j = decltype(jc)::value;
      if constexpr (j < NPV) {
        constexpr int ts = j / DT, dt = j % DT;
        ot[dt] = mfma_32x32x16<BF16>(opq[j % PF], pb[SET ^ 1][ts >> 1][ts & 1], ot[dt]);
      } else {
        constexpr int s = (j - NPV) / NTL, t = (j - NPV) % NTL;
        st[SET ^ 1][t] = mfma_32x32x16<BF16>(opq[j % PF], qf[s], s == 0 ? zero16 : st[SET ^ 1][t]);
      }
      if constexpr (j + PF < NS) {
        constexpr int n = j + PF;
        if constexpr (n < NPV) {
          opq[j % PF] = v_frag(tV, n);
        } else {
          opq[j % PF] = k_frag(tK, (n - NPV) / NTL, (n - NPV) % NTL);
        }
      }
      static_for<LPS>([&](auto lc) {
        constexpr int n = (j / LSP) * LPS + decltype(lc)::value;
        if constexpr (j % LSP == 0 && n < NL) issue_load(n, SET, k_key0, v_key0, rk, rv);
      });
      constexpr int i_lo = j * NPR / NS, i_hi = (j + 1) * NPR / NS;
      static_for<i_hi - i_lo>([&](auto dc) { weights(set_c, IntC<i_lo + decltype(dc)::value>{}, rs0, rs1); });
      __builtin_amdgcn_sched_barrier(0);
    });
    __builtin_amdgcn_s_setprio(0);
    return rs0 + rs1;
  };

  // Steps behind the last one: loads whose rows all lie behind `to` and arrive as zeros.
  auto iteration = [&](auto set_c, auto first_c, int it) {
    constexpr int SET = decltype(set_c)::value;
    const int key0 = from_kg + it * NEXT;
    wait_loads();
    __syncthreads();
    u32x4_t opq[PF];
    body_prefetch(set_c, first_c, opq);
    const bool whole = key0 + STEP - 1 <= first_key && key0 + STEP <= to;
    if ((owed != 0) | (p.softcap > 0.f) | !whole) {
      if (owed & kOwesRescale) rescale();
      if (p.softcap > 0.f) cap_scores<NTL>(st[SET], p.softcap, p.cap_c2);
      if (!whole) {
        int l = lane;  // (the row's last key is worked out here, not kept in a register over the walk)
        asm volatile("" : "+v"(l));
        int limit = to - 1;
        if (p.causal) {
          const int r = row0 + (l & 31) < rows_all ? row0 + (l & 31) : rows_all - 1;
          const int last = shift + int(divide(uint32_t(r), p.group));
          limit = last < limit ? last : limit;
        }
        mask_scores<NTL>(st[SET], limit - key0, l >> 5);
      }
      if (owed & kOwesLook) look(set_c);
    }
    need_window(vwin, kwin, key0);
    need_window(kwin, vwin, key0 + 2 * NEXT);
    float sum = body(set_c, first_c, key0 + 2 * NEXT, key0, opq);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(sum <= kGrown)) != 0, 0)) {
      owed |= kOwesLook;
      if (__builtin_amdgcn_ballot_w64(!(sum <= kRedo)) != 0) redo(set_c, sum);
    }
    l_run += sum;
  };
  if (nsteps > 0) {
    need_window(kwin, kwin, from_kg);
    {
      const i32x4_t r0 = rows_of(false, from_kg);
#pragma unroll
      for (int i = 0; i < NCH; ++i) issue_load(NCH + i, 0, from_kg, 0, r0, r0);
    }
    need_window(kwin, kwin, from_kg + NEXT);
    {
      const i32x4_t r1 = rows_of(false, from_kg + NEXT);
#pragma unroll
      for (int i = 0; i < NCH; ++i) issue_load(NCH + i, 1, from_kg + NEXT, 0, r1, r1);
    }
  }
  // (while the first tiles are on their way)
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) ot[dt] = zero16;
  if (nsteps > 0) {
    wait_loads_but<NCH>();  // K(1) may be under way
    __syncthreads();
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int t = 0; t < NTL; ++t) st[0][t] = mfma_32x32x16<BF16>(k_frag(sK, s, t), qf[s], s == 0 ? zero16 : st[0][t]);
    // (the first iteration's loads overwrite the tile that has just been read: its barrier comes first)
    iteration(IntC<0>{}, IntC<1>{}, 0);
    if (1 < nsteps) iteration(IntC<1>{}, IntC<0>{}, 1);
    for (int it = 2; it < nsteps; it += 2) {
      iteration(IntC<0>{}, IntC<0>{}, it);
      if (it + 1 < nsteps) iteration(IntC<1>{}, IntC<0>{}, it + 1);
    }
    wait_loads();
    __syncthreads();
    if (owed & kOwesRescale) rescale();
    auto drain = [&](auto set_c) {
      constexpr int SET = decltype(set_c)::value;
#pragma unroll
      for (int j = 0; j < NPV_ALL; ++j) {
        const int ts = j / DT, dt = j % DT;
        ot[dt] = mfma_32x32x16<BF16>(v_frag(sV + SET * TILE, j), pb[SET][ts >> 1][ts & 1], ot[dt]);
      }
    };
    if ((nsteps - 1) & 1) {
      drain(IntC<1>{});
    } else {
      drain(IntC<0>{});
    }
  }
  const bool several = p.causal && first_key < last_key;  // rows that attend different keys
  if constexpr (KG > 1) {
    static_assert(W * kMergeBytes<D> <= kTileLdsBytes<D, M>, "merge layout");
    __syncthreads();  // (the group's other wave may still read V)
    merge_groups<BF16, D, M, KG, PAGED>(p, u, head, u.slot, row0, rows_all, ot, m_run, l_run, several, lds_raw,
                                        kTileLdsBytes<D, M>, w * kMergeBytes<D>, kg, from, to, lane);
    return;
  }
  // (the K tiles are read by nobody any more: a wave stages its rows in a quarter of them)
  const uint32_t odd = several ? odd_rows<DT>(ot) & live_rows(rows_all - row0) : 0u;
  store_rows<BF16, D, M>(p, u, head, u.slot, row0, rows_all, ot, m_run, l_run, odd, sK + w * 32 * D, lane);
  if (odd != 0) sum_rows_again<BF16, D, M, PAGED>(p, u, head, u.slot, row0, odd, from, to, lane);
}

// Joins the parts of a row.  A wave has one token and R of its heads, 16 bytes of a part's row per lane.  Clears the rows
// behind the last sequence too.
template <int D>
constexpr int kJoinRows = 256 / D;
template <bool BF16, int D, int M>
__global__ void __launch_bounds__(256) serve_join_kernel(const ServeParams p) {
  typedef __attribute__((ext_vector_type(4))) float f32x4_t;
  constexpr int R = kJoinRows<D>, LPR = 64 / R;  // lanes per row
  const int lane = threadIdx.x & 63;
  const uint32_t id = blockIdx.x * 4u + uint32_t(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
  const int Hq = p.Hk * p.G, groups = (Hq + R - 1) / R;
  const int t = int(id / uint32_t(groups)), h = int(id - uint32_t(t) * uint32_t(groups)) * R + lane / LPR;
  if (t >= p.T) return;
  const bool behind = t >= p.cu[p.B];
  const int32_t* told = p.joins + int64_t(t) * 4;
  const int first = load_uniform(told), parts = behind ? 0 : load_uniform(told + 1), before = load_uniform(told + 2);
  if (parts == 1) return;  // written where it was computed
  const bool mine = h < Hq;
  const int d = (lane & (LPR - 1)) * 4;
  const int64_t out = int64_t(t) * Hq + h;
  if (behind) {
    if (mine) {
      *reinterpret_cast<u32x2_t*>(p.o + out * D + d) = u32x2_t{0u, 0u};
      if (p.lse != nullptr && d == 0) p.lse[out] = -INFINITY;
    }
    return;
  }
  const int head = int(divide(uint32_t(mine ? h : Hq - 1), p.group));
  const int row = (t - first) * p.G + ((mine ? h : Hq - 1) - head * p.G);
  // (a token that no sequence has, where the offsets run backwards, has been told nothing)
  if (parts < 1 || first < 0 || first > t || before < 0 || before + (int64_t(row / M) + 1) * parts > p.slots) return;
  const int64_t at = ((before + int64_t(row / M) * parts) * p.Hk + head) * M + row % M, step = int64_t(p.Hk) * M;
  float m = -INFINITY;
  for (int i = lane & (LPR - 1); i < parts; i += LPR) m = fmaxf(m, p.stats[(at + i * step) * 2]);
#pragma unroll
  for (int x = 1; x < LPR; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
  const float m_ref = m == -INFINITY ? 0.f : m;
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  for (int i0 = 0; i0 < parts; i0 += 4) {
    f32x4_t x[4];
    float w[4], lw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // (the last part again in the place of those that there are not)
      const int i = i0 + j < parts ? i0 + j : parts - 1;
      x[j] = *reinterpret_cast<const f32x4_t*>(p.sums + (at + i * step) * D + d);
      w[j] = p.stats[(at + i * step) * 2];
      lw[j] = p.stats[(at + i * step) * 2 + 1];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (i0 + j >= parts) break;
      const float f = __builtin_amdgcn_exp2f(w[j] - m_ref);
      l = __builtin_fmaf(lw[j], f, l);
#pragma unroll
      for (int k = 0; k < 4; ++k) sum[k] = __builtin_fmaf(x[j][k], f, sum[k]);
    }
  }
  if (!mine) return;
  const bool live = l > 0.f || l != l;
  const float inv = live ? 1.f / l : 0.f;
  const u32x2_t ov = {live ? pack2<BF16>(sum[0] * inv, sum[1] * inv) : 0u, live ? pack2<BF16>(sum[2] * inv, sum[3] * inv) : 0u};
  *reinterpret_cast<u32x2_t*>(p.o + out * D + d) = ov;
  if (p.lse != nullptr && d == 0) p.lse[out] = live ? (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace omni_attn
