// Norm and rotation of query and key heads, forward and backward, and the paged cache's append.
//
//   n = x * rsqrt(mean(x^2) + eps) * w         per head, in 32 bits (left out where there is no weight)
//   y_a = n_a cos - n_b sin,  y_b = n_b cos + n_a sin      for every rotating pair (a, b); the rest of the head stays
// and back, with g = R^T dy, r = rsqrt(mean(x^2) + eps), u = x r:
//   dx = r (g w - u mean(g w u)),  dw = sum over rows of g u.
// Every result is rounded once, from 32 bits.
//
// All three kernels are bound by memory: each element is read once and written once, 16 bytes per lane
// at a time.  A row (one head of one token) belongs to LPR neighbouring lanes; a lane has V pairs of it, so
// both members of a pair, their cosine, sine and weights meet in one lane and only the mean of squares crosses
// lanes.  A wave has one token (several waves share its heads where there are many): its position, sequence
// and page are the same for all lanes, and its cosines and sines are fetched once for all heads.
#include "../../include/omni_attn_gfx950.h"
#include "omni_attn_fwd_kernel.hpp"

#include <cmath>

namespace omni_attn {
namespace {

constexpr int kBlockWaves = 4;
constexpr int kRowsInFlight = 4;  // rows of a lane that are loaded before the first is worked on

typedef __attribute__((ext_vector_type(4))) float f32x4_t;

struct Heads {  // one operand: rows of D elements at a token and head
  const uint16_t* in;
  uint16_t* out;
  RowStrides in_at, out_at;  // (b, h, row); row holds the token stride
  const void* weight;        // null: no norm
  int heads;
};

struct RotaryParams {
  Heads q, k;
  const float* table;     // [table_rows, rot]: cosines, then sines
  const void* positions;  // [B, S] at pos_b, or null (append: the place in the cache)
  int64_t pos_b;
  int pos64, weight32;
  int64_t tokens;  // B * S
  int S, D, rot, table_rows;
  int lanes_per_row, waves_per_token;
  float eps, sign;  // sign -1: the inverse rotation
};

struct AppendParams {
  RotaryParams r;      // q.heads 0: no queries
  const uint16_t* v;
  RowStrides v_at;     // (h, row)
  uint16_t *k_pages, *v_pages;  // [num_pages, Hk, page, D]
  const int32_t *page_table, *kv_lens, *cu;
  int sequences, max_pages, num_pages, page_shift;
};

struct RotaryBwdParams {
  RotaryParams r;  // in: the incoming gradients, out: the outgoing ones
  const uint16_t *xq, *xk;
  RowStrides xq_at, xk_at;
  float* partial;  // [2, blocks, D]
};

template <bool BF16>
__device__ __forceinline__ float widen(uint16_t x) {
  if constexpr (BF16) {
    return __builtin_bit_cast(float, uint32_t(x) << 16);
  } else {
    return float(__builtin_bit_cast(_Float16, x));
  }
}

// V 16-bit elements in registers.
template <int V>
struct Bits {
  uint32_t w[V / 2];
};
template <int V>
__device__ __forceinline__ Bits<V> load_bits(const uint16_t* p) {
  Bits<V> r;
  if constexpr (V == 8) {
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = x[i];
  } else {
    const u32x2_t x = *reinterpret_cast<const u32x2_t*>(p);
    r.w[0] = x[0];
    r.w[1] = x[1];
  }
  return r;
}
template <int V>
__device__ __forceinline__ void store_bits(uint16_t* p, const Bits<V>& b) {
  if constexpr (V == 8) {
    *reinterpret_cast<u32x4_t*>(p) = u32x4_t{b.w[0], b.w[1], b.w[2], b.w[3]};
  } else {
    *reinterpret_cast<u32x2_t*>(p) = u32x2_t{b.w[0], b.w[1]};
  }
}

// A lane's part of a row: V pairs, as two vectors of V elements at `first` and `second`.
template <int V>
struct Part {
  int first, second, pair;  // pair: index of the first pair's cosine; -1: these do not rotate
  bool live;
};
template <int V, bool INTER>
__device__ __forceinline__ Part<V> part_of(int c, int D, int rot) {
  Part<V> p;
  const int turning = rot / 2 / V;
  p.live = c < D / 2 / V;
  if (c < turning) {
    p.pair = c * V;
    p.first = INTER ? 2 * c * V : c * V;
    p.second = INTER ? p.first + V : c * V + rot / 2;
  } else {
    p.pair = -1;
    p.first = rot + 2 * (c - turning) * V;
    p.second = p.first + V;
  }
  return p;
}
// (first, second) -> the pairs' members a and b, and back.
template <bool BF16, int V, bool INTER>
__device__ __forceinline__ void to_pairs(const Bits<V>& x, const Bits<V>& y, float (&a)[V], float (&b)[V]) {
  float f[2 * V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    f[i] = widen<BF16>(uint16_t(x.w[i / 2] >> (16 * (i & 1))));
    f[V + i] = widen<BF16>(uint16_t(y.w[i / 2] >> (16 * (i & 1))));
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    a[i] = INTER ? f[2 * i] : f[i];
    b[i] = INTER ? f[2 * i + 1] : f[V + i];
  }
}
template <bool BF16, int V, bool INTER>
__device__ __forceinline__ void from_pairs(const float (&a)[V], const float (&b)[V], Bits<V>& x, Bits<V>& y) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    if constexpr (INTER) {
      x.w[i] = pack2<BF16>(a[i], b[i]);
      y.w[i] = pack2<BF16>(a[V / 2 + i], b[V / 2 + i]);
    } else {
      x.w[i] = pack2<BF16>(a[2 * i], a[2 * i + 1]);
      y.w[i] = pack2<BF16>(b[2 * i], b[2 * i + 1]);
    }
  }
}
template <bool BF16, int V, bool INTER>
__device__ __forceinline__ void load_weight(const void* w, int weight32, const Part<V>& at, float (&a)[V], float (&b)[V]) {
  const int first = at.live ? at.first : 0, second = at.live ? at.second : 0;
#pragma unroll
  for (int i = 0; i < V; ++i) a[i] = b[i] = 1.f;
  if (w == nullptr) return;
  if (!weight32) {
    to_pairs<BF16, V, INTER>(load_bits<V>(static_cast<const uint16_t*>(w) + first),
                             load_bits<V>(static_cast<const uint16_t*>(w) + second), a, b);
    return;
  }
  const float* f = static_cast<const float*>(w);
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const f32x4_t x = *reinterpret_cast<const f32x4_t*>(f + first + i), y = *reinterpret_cast<const f32x4_t*>(f + second + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // element i + j of the first vector, and of the second
      if constexpr (INTER) {
        ((j & 1) ? b : a)[(i + j) / 2] = x[j];
        ((j & 1) ? b : a)[(V + i + j) / 2] = y[j];
      } else {
        a[i + j] = x[j];
        b[i + j] = y[j];
      }
    }
  }
}
template <int V>
__device__ __forceinline__ void load_turn(const RotaryParams& p, int64_t position, const Part<V>& at, float (&c)[V],
                                          float (&s)[V]) {
  // (a position outside the table reads its first or last row)
  const int64_t row = position < 0 ? 0 : (position < p.table_rows ? position : int64_t(p.table_rows) - 1);
  const float* t = p.table + row * p.rot;
  const int from = at.pair >= 0 ? at.pair : 0;
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    f32x4_t cosines = {1.f, 1.f, 1.f, 1.f}, sines = {0.f, 0.f, 0.f, 0.f};
    if (p.rot > 0) {
      cosines = *reinterpret_cast<const f32x4_t*>(t + from + i);
      sines = *reinterpret_cast<const f32x4_t*>(t + p.rot / 2 + from + i);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[i + j] = at.pair >= 0 ? cosines[j] : 1.f;
      s[i + j] = at.pair >= 0 ? sines[j] * p.sign : 0.f;
    }
  }
}
__device__ __forceinline__ int64_t position_of(const RotaryParams& p, int64_t index) {
  return p.pos64 ? static_cast<const int64_t*>(p.positions)[index] : int64_t(static_cast<const int32_t*>(p.positions)[index]);
}
// Sum over the lanes of a row (a power of two of neighbours).
__device__ __forceinline__ float row_sum(float x, int lanes) {
  for (int m = 1; m < lanes; m <<= 1) x += __shfl_xor(x, m);
  return x;
}

// Norm and rotation of one row's part, in place.
template <int V>
__device__ __forceinline__ void norm_turn(float (&a)[V], float (&b)[V], bool norm, const float (&wa)[V], const float (&wb)[V],
                                          const float (&c)[V], const float (&s)[V], int lanes, int D, float eps) {
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) sum = __builtin_fmaf(a[i], a[i], __builtin_fmaf(b[i], b[i], sum));
  const float r = norm ? 1.f / __builtin_sqrtf(row_sum(sum, lanes) / float(D) + eps) : 1.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float na = a[i] * r * wa[i], nb = b[i] * r * wb[i];
    a[i] = __builtin_fmaf(-nb, s[i], na * c[i]);
    b[i] = __builtin_fmaf(na, s[i], nb * c[i]);
  }
}

// Rows of q and k of one token, dealt to the row slots of the token's waves.
template <bool BF16, int V, bool INTER>
__global__ void __launch_bounds__(kBlockWaves * 64) qk_rotary_kernel(RotaryParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t wave = int64_t(blockIdx.x) * kBlockWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t token = wave / p.waves_per_token;
  if (token >= p.tokens) return;
  const int slots = 64 / p.lanes_per_row * p.waves_per_token;  // rows of the token at a time
  const int slot = int(wave - token * p.waves_per_token) * (64 / p.lanes_per_row) + lane / p.lanes_per_row;
  const int64_t b = token / p.S, s = token - b * p.S;
  const Part<V> at = part_of<V, INTER>(lane % p.lanes_per_row, p.D, p.rot);
  const uint16_t* qin = p.q.in + b * p.q.in_at.b + s * p.q.in_at.row;
  const uint16_t* kin = p.k.in + b * p.k.in_at.b + s * p.k.in_at.row;
  uint16_t* qout = p.q.out + b * p.q.out_at.b + s * p.q.out_at.row;
  uint16_t* kout = p.k.out + b * p.k.out_at.b + s * p.k.out_at.row;
  const int rows = p.q.heads + p.k.heads;
  float wqa[V], wqb[V], wka[V], wkb[V], c[V], sn[V];
  load_weight<BF16, V, INTER>(p.q.weight, p.weight32, at, wqa, wqb);
  load_weight<BF16, V, INTER>(p.k.weight, p.weight32, at, wka, wkb);
  load_turn<V>(p, position_of(p, b * p.pos_b + s), at, c, sn);
  for (int r0 = slot; r0 - slot < rows; r0 += kRowsInFlight * slots) {  // (all lanes: the sums cross them)
    Bits<V> x[kRowsInFlight], y[kRowsInFlight];
#pragma unroll
    for (int i = 0; i < kRowsInFlight; ++i) {
      const int r = r0 + i * slots;
      x[i] = y[i] = Bits<V>{};
      if (r < rows && at.live) {
        const uint16_t* in = r < p.q.heads ? qin + r * p.q.in_at.h : kin + (r - p.q.heads) * p.k.in_at.h;
        x[i] = load_bits<V>(in + at.first);
        y[i] = load_bits<V>(in + at.second);
      }
    }
#pragma unroll
    for (int i = 0; i < kRowsInFlight; ++i) {
      const int r = r0 + i * slots;
      if (r - slot >= rows) break;  // (the same for all lanes)
      const bool is_q = r < p.q.heads;
      float a[V], bb[V], wa[V], wb[V];
      to_pairs<BF16, V, INTER>(x[i], y[i], a, bb);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        wa[j] = is_q ? wqa[j] : wka[j];
        wb[j] = is_q ? wqb[j] : wkb[j];
      }
      norm_turn<V>(a, bb, (is_q ? p.q.weight : p.k.weight) != nullptr, wa, wb, c, sn, p.lanes_per_row, p.D, p.eps);
      if (r < rows && at.live) {
        uint16_t* out = is_q ? qout + r * p.q.out_at.h : kout + (r - p.q.heads) * p.k.out_at.h;
        from_pairs<BF16, V, INTER>(a, bb, x[i], y[i]);
        store_bits<V>(out + at.first, x[i]);
        store_bits<V>(out + at.second, y[i]);
      }
    }
  }
}

// The same with keys and values going to their sequence's pages.  Rows: queries, keys, values.
template <bool BF16, int V, bool INTER>
__global__ void __launch_bounds__(kBlockWaves * 64) cache_append_kernel(AppendParams ap) {
  const RotaryParams& p = ap.r;
  const int lane = threadIdx.x & 63;
  const int64_t wave = int64_t(blockIdx.x) * kBlockWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t token = wave / p.waves_per_token;
  if (token >= p.tokens) return;
  const int slots = 64 / p.lanes_per_row * p.waves_per_token;
  const int slot = int(wave - token * p.waves_per_token) * (64 / p.lanes_per_row) + lane / p.lanes_per_row;
  const Part<V> at = part_of<V, INTER>(lane % p.lanes_per_row, p.D, p.rot);
  const uint16_t* qin = p.q.in + token * p.q.in_at.row;
  const uint16_t* kin = p.k.in + token * p.k.in_at.row;
  const uint16_t* vin = ap.v + token * ap.v_at.row;
  uint16_t* qout = p.q.out + token * p.q.out_at.row;
  const int qk = p.q.heads + p.k.heads, rows = qk + p.k.heads;
  bool owned = false;
  Bits<V> x[kRowsInFlight], y[kRowsInFlight];
  auto request = [&](int r0) {
#pragma unroll
    for (int i = 0; i < kRowsInFlight; ++i) {
      const int r = r0 + i * slots;
      x[i] = y[i] = Bits<V>{};
      if (r < rows && at.live) {
        const uint16_t* in = r < p.q.heads ? qin + r * p.q.in_at.h
                             : r < qk      ? kin + (r - p.q.heads) * p.k.in_at.h
                                           : vin + (r - qk) * ap.v_at.h;
        x[i] = load_bits<V>(in + at.first);
        y[i] = load_bits<V>(in + at.second);
      }
    }
  };
  // The token's sequence: as many as end at or before it come first.  A lane looks at every per-th end, then at those
  // between.  (With the rows asked for before the look-up, behind the first ends: 12 prompts of 11000 tokens 45.2 us for 42.4,
  // single tokens the same.)
  const int per = (ap.sequences + 63) / 64;
  const int64_t last = int64_t(lane + 1) * per;
  const int end = ap.cu[last <= ap.sequences ? last : 0];
  int b = __builtin_popcountll(__builtin_amdgcn_ballot_w64(last <= ap.sequences && end <= token)) * per;
  for (int j0 = 0, from = b; per > 1 && j0 < per && from + j0 < ap.sequences; j0 += 64) {
    const int j = from + j0 + lane;
    const bool in = j < ap.sequences && j0 + lane < per;
    b += __builtin_popcountll(__builtin_amdgcn_ballot_w64(in && ap.cu[1 + (in ? j : 0)] <= token));
  }
  int64_t position = -1;
  uint16_t *krow = nullptr, *vrow = nullptr;
  if (b < ap.sequences) {
    const int first = b == 0 ? 0 : load_uniform(ap.cu + b), behind = load_uniform(ap.cu + b + 1);
    const int64_t keys = load_uniform(ap.kv_lens + b);
    if (token >= first && token < behind) {
      owned = true;
      position = keys - behind + token;
      const int64_t in_table = position >> ap.page_shift;
      if (position >= 0 && in_table < ap.max_pages) {
        const int page = load_uniform(ap.page_table + int64_t(b) * ap.max_pages + in_table);
        if (page >= 0 && page < ap.num_pages) {
          const int64_t row = ((int64_t(page) * p.k.heads) << ap.page_shift) + (position & ((1 << ap.page_shift) - 1));
          krow = ap.k_pages + row * p.D;
          vrow = ap.v_pages + row * p.D;
        }
      }
    }
  }
  const int64_t head_step = int64_t(p.D) << ap.page_shift;
  float wqa[V], wqb[V], wka[V], wkb[V], c[V], sn[V];
  load_weight<BF16, V, INTER>(p.q.weight, p.weight32, at, wqa, wqb);
  load_weight<BF16, V, INTER>(p.k.weight, p.weight32, at, wka, wkb);
  load_turn<V>(p, p.positions ? position_of(p, token) : position, at, c, sn);
  for (int r0 = slot; r0 - slot < rows; r0 += kRowsInFlight * slots) {
    request(r0);
#pragma unroll
    for (int i = 0; i < kRowsInFlight; ++i) {
      const int r = r0 + i * slots;
      if (r - slot >= rows) break;
      const bool is_q = r < p.q.heads;
      float a[V], bb[V], wa[V], wb[V];
      to_pairs<BF16, V, INTER>(x[i], y[i], a, bb);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        wa[j] = is_q ? wqa[j] : wka[j];
        wb[j] = is_q ? wqb[j] : wkb[j];
      }
      norm_turn<V>(a, bb, (is_q ? p.q.weight : p.k.weight) != nullptr, wa, wb, c, sn, p.lanes_per_row, p.D, p.eps);
      if (r >= rows || !at.live) continue;
      uint16_t* out = is_q   ? qout + r * p.q.out_at.h
                      : !krow ? nullptr
                      : r < qk ? krow + (r - p.q.heads) * head_step
                               : vrow + (r - qk) * head_step;
      if (out == nullptr) continue;  // a token without a place in the cache
      Bits<V> ox, oy;
      from_pairs<BF16, V, INTER>(a, bb, ox, oy);
      if (r >= qk) {  // values go through bit for bit
        ox = x[i];
        oy = y[i];
      } else if (!owned) {  // behind the last sequence: zeros
        ox = oy = Bits<V>{};
      }
      store_bits<V>(out + at.first, ox);
      store_bits<V>(out + at.second, oy);
    }
  }
}

constexpr int kBackV = 4;  // (of 8: 144 registers and three waves per SIMD for 88 and five, 53 us for 51)

// Gradients of one side: queries (blockIdx.y 0) or keys.  A wave walks the tokens, several at a time where there are
// fewer heads than it has rows; its lanes keep their dimensions' sums of dw in registers, a block's four waves add theirs
// up in LDS and write one row of `partial`.  (Both sides in one wave: weights and sums of both, 171 registers and two
// waves per SIMD; 2 x 4096 tokens, 32 / 8 heads, D=128: 67 us, 51 so, 4.9 TB/s.)
template <bool BF16, int V, bool INTER>
__global__ void __launch_bounds__(kBlockWaves * 64) qk_rotary_bwd_kernel(RotaryBwdParams bp) {
  constexpr int kRows = 2;
  const RotaryParams& p = bp.r;
  const bool is_k = blockIdx.y != 0;
  const Heads& io = is_k ? p.k : p.q;
  const uint16_t* xs = is_k ? bp.xk : bp.xq;
  const RowStrides& x_at = is_k ? bp.xk_at : bp.xq_at;
  const bool norm = io.weight != nullptr;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slots = 64 / p.lanes_per_row, slot = lane / p.lanes_per_row;
  int head_slots = 1;  // rows of a token that a wave has at a time
  while (head_slots < slots && head_slots < io.heads) head_slots <<= 1;
  const int tokens_at_once = slots / head_slots;
  const Part<V> at = part_of<V, INTER>(lane % p.lanes_per_row, p.D, p.rot);
  float wa[V], wb[V];
  load_weight<BF16, V, INTER>(io.weight, p.weight32, at, wa, wb);
  float gw[2][V] = {};
  const int64_t stride = int64_t(gridDim.x) * kBlockWaves * tokens_at_once;
  for (int64_t t0 = (int64_t(blockIdx.x) * kBlockWaves + wv) * tokens_at_once; t0 < p.tokens; t0 += stride) {
    const int64_t mine = t0 + slot / head_slots;
    const bool has = mine < p.tokens && at.live;
    const int64_t token = mine < p.tokens ? mine : p.tokens - 1;
    const int64_t b = token / p.S, s = token - b * p.S;
    const uint16_t* in = io.in + b * io.in_at.b + s * io.in_at.row;
    const uint16_t* xin = xs + b * x_at.b + s * x_at.row;
    uint16_t* out = io.out + b * io.out_at.b + s * io.out_at.row;
    float c[V], sn[V];
    load_turn<V>(p, position_of(p, b * p.pos_b + s), at, c, sn);
    for (int h0 = 0; h0 < io.heads; h0 += kRows * head_slots) {
      Bits<V> dx[kRows], dy[kRows], x[kRows], y[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int h = h0 + i * head_slots + (slot & (head_slots - 1));
        dx[i] = dy[i] = x[i] = y[i] = Bits<V>{};
        if (h < io.heads && has) {
          dx[i] = load_bits<V>(in + h * io.in_at.h + at.first);
          dy[i] = load_bits<V>(in + h * io.in_at.h + at.second);
          if (norm) {
            x[i] = load_bits<V>(xin + h * x_at.h + at.first);
            y[i] = load_bits<V>(xin + h * x_at.h + at.second);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        if (h0 + i * head_slots >= io.heads) break;  // (the same for all lanes: the sums cross them)
        const int h = h0 + i * head_slots + (slot & (head_slots - 1));
        const bool row = h < io.heads && has;
        float da[V], db[V];
        to_pairs<BF16, V, INTER>(dx[i], dy[i], da, db);
#pragma unroll
        for (int j = 0; j < V; ++j) {  // (s carries the sign of the inverse rotation)
          const float ga = __builtin_fmaf(-db[j], sn[j], da[j] * c[j]), gb = __builtin_fmaf(da[j], sn[j], db[j] * c[j]);
          da[j] = ga;
          db[j] = gb;
        }
        if (norm) {
          float a[V], bb[V], squares = 0.f, dots = 0.f;
          to_pairs<BF16, V, INTER>(x[i], y[i], a, bb);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            squares = __builtin_fmaf(a[j], a[j], __builtin_fmaf(bb[j], bb[j], squares));
            dots = __builtin_fmaf(da[j] * wa[j], a[j], __builtin_fmaf(db[j] * wb[j], bb[j], dots));
          }
          squares = row_sum(squares, p.lanes_per_row);
          dots = row_sum(dots, p.lanes_per_row);
          const float rs = 1.f / __builtin_sqrtf(squares / float(p.D) + p.eps);
          const float pull = dots * rs * rs / float(p.D);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            gw[0][j] += row ? da[j] * a[j] * rs : 0.f;
            gw[1][j] += row ? db[j] * bb[j] * rs : 0.f;
            da[j] = rs * __builtin_fmaf(-a[j], pull, da[j] * wa[j]);
            db[j] = rs * __builtin_fmaf(-bb[j], pull, db[j] * wb[j]);
          }
        }
        if (row) {
          from_pairs<BF16, V, INTER>(da, db, dx[i], dy[i]);
          store_bits<V>(out + h * io.out_at.h + at.first, dx[i]);
          store_bits<V>(out + h * io.out_at.h + at.second, dy[i]);
        }
      }
    }
  }
  if (bp.partial == nullptr) return;
  __shared__ float sums[kBlockWaves][256];
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      for (int m = p.lanes_per_row; m < 64; m <<= 1) gw[h][j] += __shfl_xor(gw[h][j], m);
  if (slot == 0 && at.live) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int ia = INTER ? at.first + 2 * j : at.first + j, ib = INTER ? ia + 1 : at.second + j;
      sums[wv][ia] = gw[0][j];
      sums[wv][ib] = gw[1][j];
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < p.D; d += kBlockWaves * 64) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kBlockWaves; ++w) t += sums[w][d];
    bp.partial[(int64_t(blockIdx.y) * gridDim.x + blockIdx.x) * p.D + d] = t;
  }
}

// dw of 16 dimensions per block: 16 row lanes each, in 64 bits, added up in a fixed order.  blockIdx.y: the side.
__global__ void __launch_bounds__(256) rotary_weight_grad_kernel(const float* partial, int blocks, int D, void* dwq,
                                                                 void* dwk, int weight32, int bf16) {
  __shared__ double sums[16][17];
  void* out = blockIdx.y ? dwk : dwq;
  if (out == nullptr) return;
  const int part = threadIdx.x >> 4, column = blockIdx.x * 16 + (threadIdx.x & 15);
  double t = 0;
  if (column < D) {
#pragma unroll 8
    for (int i = part; i < blocks; i += 16) t += double(partial[(int64_t(blockIdx.y) * blocks + i) * D + column]);
  }
  sums[part][threadIdx.x & 15] = t;
  __syncthreads();
  if (part != 0 || column >= D) return;
  for (int i = 1; i < 16; ++i) t += sums[i][threadIdx.x & 15];
  if (weight32) {
    static_cast<float*>(out)[column] = float(t);
  } else if (bf16) {
    static_cast<uint16_t*>(out)[column] = __builtin_bit_cast(uint16_t, __bf16(float(t)));
  } else {
    static_cast<uint16_t*>(out)[column] = __builtin_bit_cast(uint16_t, _Float16(float(t)));
  }
}

// ---- host side --------------------------------------------------------------------------------------

bool misaligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

int check_heads(int D, int rot, int Hq, int Hk, int table_rows, float eps, int dtype) {
  if (dtype != OMNI_ATTN_DTYPE_F16 && dtype != OMNI_ATTN_DTYPE_BF16) return OMNI_ATTN_ERR_UNSUPPORTED_DTYPE;
  if (D < 8 || D > 256 || D % 8 != 0) return OMNI_ATTN_ERR_UNSUPPORTED_HEAD_DIM;
  if (rot < 0 || rot > D || rot % 8 != 0 || Hq < 0 || Hk < 1 || Hq > 65536 || Hk > 65536 || (rot > 0 && table_rows < 1) ||
      !(eps >= 0.f) || std::isinf(eps))
    return OMNI_ATTN_ERR_BAD_SHAPE;
  return OMNI_ATTN_OK;
}
// 8-byte pieces of every operand; strides that keep them aligned.
int check_rows(const void* p, const omni_attn_strides& at) {
  if (misaligned(p, 8) || at.batch % 4 != 0 || at.head % 4 != 0 || at.row % 4 != 0) return OMNI_ATTN_ERR_MISALIGNED;
  if (at.batch < 0 || at.head < 0 || at.row < 0) return OMNI_ATTN_ERR_BAD_SHAPE;
  if (at.row > 0x7fffffffLL) return OMNI_ATTN_ERR_TOO_LARGE;
  return OMNI_ATTN_OK;
}
bool wide_rows(const void* p, const omni_attn_strides& at) {
  return !misaligned(p, 16) && at.batch % 8 == 0 && at.head % 8 == 0 && at.row % 8 == 0;
}
RowStrides strides(const omni_attn_strides& at) { return {at.batch, at.head, uint32_t(at.row)}; }

// Vectors of 8 elements (16 bytes) where every operand and both parts of a head are made of them, else of 4; heads of
// 32 dimensions too, whose two lanes per row would leave a wave with 32 rows of one token.
int vector_width(bool wide, int D, int rot) { return wide && D > 32 && rot % 16 == 0 && (D - rot) % 16 == 0 ? 8 : 4; }

void deal_rows(RotaryParams& p, int V, int rows) {
  const int parts = p.D / 2 / V;
  p.lanes_per_row = 1;
  while (p.lanes_per_row < parts) p.lanes_per_row <<= 1;
  const int per_wave = 64 / p.lanes_per_row;
  const int most = (rows + per_wave - 1) / per_wave;
  const int least = (rows + kRowsInFlight * per_wave - 1) / (kRowsInFlight * per_wave);
  // A lane has up to four rows; fewer, in more waves, where a launch would not give every SIMD two waves.
  p.waves_per_token = p.tokens * least >= 2048 ? least : most;
}

template <bool BF16, int V, bool INTER>
void launch_forward(const RotaryParams& p, unsigned blocks, hipStream_t stream) {
  hipLaunchKernelGGL((qk_rotary_kernel<BF16, V, INTER>), dim3(blocks), dim3(kBlockWaves * 64), 0, stream, p);
}
template <bool BF16, int V, bool INTER>
void launch_append(const AppendParams& p, unsigned blocks, hipStream_t stream) {
  hipLaunchKernelGGL((cache_append_kernel<BF16, V, INTER>), dim3(blocks), dim3(kBlockWaves * 64), 0, stream, p);
}
template <bool BF16, bool INTER>
void launch_backward(const RotaryBwdParams& p, unsigned blocks, hipStream_t stream) {
  hipLaunchKernelGGL((qk_rotary_bwd_kernel<BF16, kBackV, INTER>), dim3(blocks, 2), dim3(kBlockWaves * 64), 0, stream, p);
}
#define OMNI_ROTARY_INSTANCE(launch, bf16, V, inter, ...)                                                   \
  do {                                                                                                      \
    if (bf16) {                                                                                             \
      if ((V) == 8) (inter) ? launch<true, 8, true>(__VA_ARGS__) : launch<true, 8, false>(__VA_ARGS__);     \
      else (inter) ? launch<true, 4, true>(__VA_ARGS__) : launch<true, 4, false>(__VA_ARGS__);              \
    } else {                                                                                                \
      if ((V) == 8) (inter) ? launch<false, 8, true>(__VA_ARGS__) : launch<false, 8, false>(__VA_ARGS__);   \
      else (inter) ? launch<false, 4, true>(__VA_ARGS__) : launch<false, 4, false>(__VA_ARGS__);            \
    }                                                                                                       \
  } while (0)

int launched() {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return OMNI_ATTN_OK;
  record_hip_error(int(e));
  return OMNI_ATTN_ERR_LAUNCH;
}

// Blocks of the backward's first launch, and so rows of its partial sums.
int backward_blocks(long long tokens) {
  const long long blocks = (tokens + kBlockWaves - 1) / kBlockWaves;
  return int(blocks < 768 ? blocks : 768);
}

}  // namespace
}  // namespace omni_attn

extern "C" int omni_attn_qk_rotary_gfx950(const void* q, const void* k, omni_attn_strides q_at, omni_attn_strides k_at,
                                          void* q_out, void* k_out, omni_attn_strides q_out_at,
                                          omni_attn_strides k_out_at, const float* table, const void* positions,
                                          int64_t positions_batch, int positions_64, const void* q_weight_or_null,
                                          const void* k_weight_or_null, int weights_f32, int B, int S, int Hq, int Hk,
                                          int D, int rotary_dim, int table_rows, float eps, int interleaved, int dtype,
                                          void* stream) {
  using namespace omni_attn;
  if (!q || !k || !q_out || !k_out || !table || !positions) return OMNI_ATTN_ERR_NULL_POINTER;
  if (const int rc = check_heads(D, rotary_dim, Hq, Hk, table_rows, eps, dtype)) return rc;
  if (B <= 0 || S <= 0 || Hq < 1 || positions_batch < 0) return OMNI_ATTN_ERR_BAD_SHAPE;
  if (misaligned(table, 16) || misaligned(positions, positions_64 ? 8 : 4)) return OMNI_ATTN_ERR_MISALIGNED;
  for (const void* w : {q_weight_or_null, k_weight_or_null})
    if (misaligned(w, 16)) return OMNI_ATTN_ERR_MISALIGNED;
  bool wide = true;
  const void* ptrs[4] = {q, k, q_out, k_out};
  const omni_attn_strides* ats[4] = {&q_at, &k_at, &q_out_at, &k_out_at};
  for (int i = 0; i < 4; ++i) {
    if (const int rc = check_rows(ptrs[i], *ats[i])) return rc;
    wide = wide && wide_rows(ptrs[i], *ats[i]);
  }
  RotaryParams p{};
  p.q = {static_cast<const uint16_t*>(q), static_cast<uint16_t*>(q_out), strides(q_at), strides(q_out_at), q_weight_or_null, Hq};
  p.k = {static_cast<const uint16_t*>(k), static_cast<uint16_t*>(k_out), strides(k_at), strides(k_out_at), k_weight_or_null, Hk};
  p.table = table;
  p.positions = positions;
  p.pos_b = positions_batch;
  p.pos64 = positions_64;
  p.weight32 = weights_f32;
  p.tokens = int64_t(B) * S;
  p.S = S;
  p.D = D;
  p.rot = rotary_dim;
  p.table_rows = table_rows;
  p.eps = eps;
  p.sign = 1.f;
  const int V = vector_width(wide, D, rotary_dim);
  deal_rows(p, V, Hq + Hk);
  const long long blocks = (p.tokens * p.waves_per_token + kBlockWaves - 1) / kBlockWaves;
  if (blocks > 0x7fffffffLL) return OMNI_ATTN_ERR_TOO_LARGE;
  OMNI_ROTARY_INSTANCE(launch_forward, dtype == OMNI_ATTN_DTYPE_BF16, V, interleaved, p, unsigned(blocks),
                       static_cast<hipStream_t>(stream));
  return launched();
}

extern "C" size_t omni_attn_qk_rotary_bwd_workspace_bytes(int B, int S, int D) {
  if (B <= 0 || S <= 0 || D <= 0) return 0;
  return size_t(omni_attn::backward_blocks((long long)B * S)) * 2 * size_t(D) * sizeof(float);
}

extern "C" int omni_attn_qk_rotary_bwd_gfx950(
    const void* dq_out, const void* dk_out, const void* q, const void* k, omni_attn_strides dq_out_at,
    omni_attn_strides dk_out_at, omni_attn_strides q_at, omni_attn_strides k_at, void* dq, void* dk,
    omni_attn_strides dq_at, omni_attn_strides dk_at, void* dq_weight_or_null, void* dk_weight_or_null,
    const float* table, const void* positions, int64_t positions_batch, int positions_64, const void* q_weight_or_null,
    const void* k_weight_or_null, int weights_f32, void* workspace, size_t workspace_bytes, int B, int S, int Hq, int Hk,
    int D, int rotary_dim, int table_rows, float eps, int interleaved, int dtype, void* stream) {
  using namespace omni_attn;
  if (!dq_out || !dk_out || !dq || !dk || !table || !positions) return OMNI_ATTN_ERR_NULL_POINTER;
  if ((q_weight_or_null && !q) || (k_weight_or_null && !k)) return OMNI_ATTN_ERR_NULL_POINTER;
  if ((dq_weight_or_null && !q_weight_or_null) || (dk_weight_or_null && !k_weight_or_null)) return OMNI_ATTN_ERR_NULL_POINTER;
  if (const int rc = check_heads(D, rotary_dim, Hq, Hk, table_rows, eps, dtype)) return rc;
  if (B <= 0 || S <= 0 || Hq < 1 || positions_batch < 0) return OMNI_ATTN_ERR_BAD_SHAPE;
  if (misaligned(table, 16) || misaligned(positions, positions_64 ? 8 : 4) || misaligned(workspace, 4))
    return OMNI_ATTN_ERR_MISALIGNED;
  for (const void* w : {q_weight_or_null, k_weight_or_null, static_cast<const void*>(dq_weight_or_null),
                        static_cast<const void*>(dk_weight_or_null)})
    if (misaligned(w, 16)) return OMNI_ATTN_ERR_MISALIGNED;
  const bool weights = dq_weight_or_null || dk_weight_or_null;
  if (weights && (!workspace || workspace_bytes < omni_attn_qk_rotary_bwd_workspace_bytes(B, S, D)))
    return OMNI_ATTN_ERR_WORKSPACE;
  bool wide = true;
  const void* ptrs[6] = {dq_out, dk_out, dq, dk, q_weight_or_null ? q : nullptr, k_weight_or_null ? k : nullptr};
  const omni_attn_strides* ats[6] = {&dq_out_at, &dk_out_at, &dq_at, &dk_at, &q_at, &k_at};
  for (int i = 0; i < 6; ++i) {
    if (ptrs[i] == nullptr) continue;
    if (const int rc = check_rows(ptrs[i], *ats[i])) return rc;
    wide = wide && wide_rows(ptrs[i], *ats[i]);
  }
  RotaryBwdParams bp{};
  RotaryParams& p = bp.r;
  p.q = {static_cast<const uint16_t*>(dq_out), static_cast<uint16_t*>(dq), strides(dq_out_at), strides(dq_at), q_weight_or_null, Hq};
  p.k = {static_cast<const uint16_t*>(dk_out), static_cast<uint16_t*>(dk), strides(dk_out_at), strides(dk_at), k_weight_or_null, Hk};
  bp.xq = static_cast<const uint16_t*>(q);
  bp.xk = static_cast<const uint16_t*>(k);
  bp.xq_at = strides(q_at);
  bp.xk_at = strides(k_at);
  bp.partial = weights ? static_cast<float*>(workspace) : nullptr;
  p.table = table;
  p.positions = positions;
  p.pos_b = positions_batch;
  p.pos64 = positions_64;
  p.weight32 = weights_f32;
  p.tokens = int64_t(B) * S;
  p.S = S;
  p.D = D;
  p.rot = rotary_dim;
  p.table_rows = table_rows;
  p.eps = eps;
  p.sign = -1.f;
  const bool turn_only = !q_weight_or_null && !k_weight_or_null;
  const int V = turn_only ? vector_width(wide, D, rotary_dim) : kBackV;
  const bool bf16 = dtype == OMNI_ATTN_DTYPE_BF16;
  deal_rows(p, V, Hq + Hk);
  if (turn_only) {  // the inverse rotation alone
    const long long blocks = (p.tokens * p.waves_per_token + kBlockWaves - 1) / kBlockWaves;
    if (blocks > 0x7fffffffLL) return OMNI_ATTN_ERR_TOO_LARGE;
    OMNI_ROTARY_INSTANCE(launch_forward, bf16, V, interleaved, p, unsigned(blocks), static_cast<hipStream_t>(stream));
    return launched();
  }
  const int blocks = backward_blocks(p.tokens);
  (bf16 ? (interleaved ? launch_backward<true, true> : launch_backward<true, false>)
        : (interleaved ? launch_backward<false, true> : launch_backward<false, false>))(bp, unsigned(blocks), static_cast<hipStream_t>(stream));
  if (const int rc = launched()) return rc;
  if (!weights) return OMNI_ATTN_OK;
  hipLaunchKernelGGL(rotary_weight_grad_kernel, dim3((D + 15) / 16, 2), dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const float*>(workspace), blocks, D, dq_weight_or_null, dk_weight_or_null, weights_f32,
                     int(bf16));
  return launched();
}

extern "C" int omni_attn_cache_append_gfx950(
    const void* q_or_null, const void* k, const void* v, omni_attn_strides q_at, omni_attn_strides k_at,
    omni_attn_strides v_at, void* q_out_or_null, omni_attn_strides q_out_at, void* k_pages, void* v_pages,
    const int32_t* page_table, const int32_t* kv_lens, const int32_t* cu_seqlens, const float* table_or_null,
    const void* positions_or_null, int positions_64, const void* q_weight_or_null, const void* k_weight_or_null,
    int weights_f32, int tokens, int sequences, int Hq, int Hk, int D, int num_pages, int page_size, int max_pages,
    int rotary_dim, int table_rows, float eps, int interleaved, int dtype, void* stream) {
  using namespace omni_attn;
  if (!k || !v || !k_pages || !v_pages || !page_table || !kv_lens || !cu_seqlens || (rotary_dim > 0 && !table_or_null) ||
      (!q_or_null != !q_out_or_null))
    return OMNI_ATTN_ERR_NULL_POINTER;
  if (const int rc = check_heads(D, rotary_dim, Hq, Hk, table_rows, eps, dtype)) return rc;
  if (tokens <= 0 || sequences <= 0 || num_pages <= 0 || max_pages <= 0 || page_size < 1 ||
      (page_size & (page_size - 1)) != 0 || (q_or_null != nullptr) != (Hq > 0))
    return OMNI_ATTN_ERR_BAD_SHAPE;
  if (misaligned(table_or_null, 16) || misaligned(positions_or_null, positions_64 ? 8 : 4) || misaligned(page_table, 4) ||
      misaligned(kv_lens, 4) || misaligned(cu_seqlens, 4) || misaligned(k_pages, 8) || misaligned(v_pages, 8))
    return OMNI_ATTN_ERR_MISALIGNED;
  for (const void* w : {q_weight_or_null, k_weight_or_null})
    if (misaligned(w, 16)) return OMNI_ATTN_ERR_MISALIGNED;
  bool wide = !misaligned(k_pages, 16) && !misaligned(v_pages, 16);
  const void* ptrs[4] = {k, v, q_or_null, q_out_or_null};
  const omni_attn_strides* ats[4] = {&k_at, &v_at, &q_at, &q_out_at};
  for (int i = 0; i < 4; ++i) {
    if (ptrs[i] == nullptr) continue;
    if (const int rc = check_rows(ptrs[i], *ats[i])) return rc;
    wide = wide && wide_rows(ptrs[i], *ats[i]);
  }
  {  // (a row would get the key and the value of a token, in any order)
    const uintptr_t k0 = reinterpret_cast<uintptr_t>(k_pages), v0 = reinterpret_cast<uintptr_t>(v_pages);
    const uint64_t bytes = uint64_t(num_pages) * uint64_t(Hk) * uint64_t(page_size) * uint64_t(D) * 2;
    if ((k0 > v0 ? k0 - v0 : v0 - k0) < bytes) return OMNI_ATTN_ERR_BAD_SHAPE;
  }
  AppendParams ap{};
  RotaryParams& p = ap.r;
  p.q = {static_cast<const uint16_t*>(q_or_null), static_cast<uint16_t*>(q_out_or_null), strides(q_at), strides(q_out_at), q_weight_or_null, Hq};
  p.k = {static_cast<const uint16_t*>(k), nullptr, strides(k_at), {}, k_weight_or_null, Hk};
  p.table = table_or_null;
  p.positions = positions_or_null;
  p.pos64 = positions_64;
  p.weight32 = weights_f32;
  p.tokens = tokens;
  p.S = tokens;
  p.D = D;
  p.rot = rotary_dim;
  p.table_rows = table_rows;
  p.eps = eps;
  p.sign = 1.f;
  ap.v = static_cast<const uint16_t*>(v);
  ap.v_at = strides(v_at);
  ap.k_pages = static_cast<uint16_t*>(k_pages);
  ap.v_pages = static_cast<uint16_t*>(v_pages);
  ap.page_table = page_table;
  ap.kv_lens = kv_lens;
  ap.cu = cu_seqlens;
  ap.sequences = sequences;
  ap.max_pages = max_pages;
  ap.num_pages = num_pages;
  ap.page_shift = __builtin_ctz(unsigned(page_size));
  const int V = vector_width(wide, D, rotary_dim);
  deal_rows(p, V, Hq + 2 * Hk);
  const long long blocks = (p.tokens * p.waves_per_token + kBlockWaves - 1) / kBlockWaves;
  if (blocks > 0x7fffffffLL) return OMNI_ATTN_ERR_TOO_LARGE;
  OMNI_ROTARY_INSTANCE(launch_append, dtype == OMNI_ATTN_DTYPE_BF16, V, interleaved, ap, unsigned(blocks),
                       static_cast<hipStream_t>(stream));
  return launched();
}
