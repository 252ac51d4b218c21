// Gradients of the attention of packed sequences over their own keys (omni_attn_serving_kernel.hpp).  With
//   P_ij = exp(x_ij - LSE_i),  x = cap(q k / sqrt(D)),  delta_i = sum_d dO_id O_id:
//   dV_j = sum_i P_ij dO_i,  dS_ij = P_ij (dO_i . v_j - delta_i) dx/d(q k / sqrt(D)),
//   dQ_i = sum_j dS_ij k_j / sqrt(D),  dK_j = sum_i dS_ij q_i / sqrt(D).
// A row i is a token and a head of the group, as in the forward, so the sums of dK and dV over the heads that share a key
// head are part of the walk over rows, and nothing is added up across workgroups: same bits every time.
//
// Two kernels.  dQ: a tile of 128 rows walks its keys; a lane owns a row, S^T = K Q^T and dP^T = V dO^T start from the
// rows' offsets (-LSE, -delta), dS^T goes as the B operand into dQ^T += K^T dS^T with K read transposed from the same
// tile.  It leaves delta for the other kernel.  dK and dV: a tile of 128 keys walks the rows that attend it; a lane owns a
// key.  Tiles of 64 keys (rows) come a step ahead by direct loads, one barrier per step; two workgroups share a compute
// unit, and the vector work of one runs under the products of the other.  P and dS are rounded to 16 bits for the second
// products (half a step of each weight, as in the forward); everything else is 32 bits.
#pragma once

#include "omni_attn_bwd_kernel.hpp"
#include "omni_attn_serving_kernel.hpp"

namespace omni_attn {

struct ServeBwdParams {
  ServeParams s;           // (dK and dV: G 1, so that tiles are of keys)
  const uint16_t* dout;    // [T, Hq, D] at dout_row, dout_head
  int64_t dout_row, dout_head;
  const uint16_t* out;     // [T, Hq, D]
  const float* lse;        // [T, Hq]
  float* delta;            // [T, Hq]
  uint16_t *dq, *dk, *dv;  // contiguous
  int G;
  FastDiv group;
  float scale, cap_l2;     // 1 / sqrt(D); cap log2(e)
};

template <int D>
constexpr size_t kServeDqLdsBytes = size_t(2) * 2 * kStepKeys * D * 2;
// At head_dim 128 the lanes' keys leave no registers for their values (77 of them were spilled): a wave's V lies in LDS,
// and steps of 32 rows make room for it there.
template <int D>
constexpr int kDkdvStep = D == 128 ? 32 : 64;
template <int D>
constexpr size_t kDkdvGroupBytes = size_t(2) * (2 * kDkdvStep<D> * D * 2 + 2 * kDkdvStep<D> * 4);  // two sets of tiles
template <int D, int KG>
constexpr size_t kServeDkdvLdsBytes = KG * kDkdvGroupBytes<D> + (D == 128 ? 128 * D * 2 : 0);

// 32 rows of a wave, transposed accumulators x factor, as whole rows; at(row): where a row goes, null: nowhere.
template <bool BF16, int D, class At>
__device__ __forceinline__ void serve_store_grad(const f32x16_t (&acc)[D / 32], float factor, uint16_t* stage, int lane, At&& at) {
  constexpr int CPR = D / 8, RPS = 64 / CPR;
  const int g = lane >> 5, c = lane & 31;
  static_for<D / 8>([&](auto ic) {
    constexpr int dt = decltype(ic)::value / 4, r4 = decltype(ic)::value % 4;
    const u32x2_t ov = {pack2<BF16>(acc[dt][4 * r4 + 0] * factor, acc[dt][4 * r4 + 1] * factor),
                        pack2<BF16>(acc[dt][4 * r4 + 2] * factor, acc[dt][4 * r4 + 3] * factor)};
    *reinterpret_cast<u32x2_t*>(stage + c * D + ((4 * dt + r4) ^ k_swizzle<D>(c)) * 8 + 4 * g) = ov;
  });
  const int pch = lane % CPR;
#pragma unroll
  for (int i = 0; i < 32 / RPS; ++i) {
    const int row = i * RPS + lane / CPR;
    const u32x4_t val = *reinterpret_cast<const u32x4_t*>(stage + row * D + pch * 8);
    uint16_t* to = at(row);
    if (to != nullptr) *reinterpret_cast<u32x4_t*>(to + (pch ^ k_swizzle<D>(row)) * 8) = val;
  }
}

template <bool BF16, int D, bool CAP>
__global__ void __launch_bounds__(256, 2) serve_dq_kernel(const ServeBwdParams b) {
  constexpr int M = 128, STEP = kStepKeys, KS = D / 16, DT = D / 32, TILE = STEP * D;
  const ServeParams& p = b.s;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
  const uint32_t lds = lds_offset_of(lds_raw);  // [2 sets][K, V][TILE]
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, c = lane & 31;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  int head, rank;
  deal_head(p, blockIdx.x, head, rank);
  if (rank >= p.units) return;
  const Unit u = find_tile<M>(p, rank, lane);
  if (!u.found) {
    clear_rows<D>(p, head, rank, u.step0, p.units, tid, 256);  // (p.o is dQ here)
    return;
  }
  const int rows_all = u.seq.n * p.G, row0 = u.tile * M + 32 * w;
  const int row = row0 + c < rows_all ? row0 + c : rows_all - 1;
  const int token = int(divide(uint32_t(row), p.group));
  const int last_row = u.tile * M + M < rows_all ? u.tile * M + M - 1 : rows_all - 1;
  const int to = __builtin_amdgcn_readfirstlane(p.causal ? int(divide(uint32_t(last_row), p.group)) + 1 : u.seq.n);
  const int first_row = row0 < rows_all ? row0 : rows_all - 1;
  const int first_key = __builtin_amdgcn_readfirstlane(p.causal ? int(divide(uint32_t(first_row), p.group)) : u.seq.n - 1);
  const int limit = p.causal ? token : u.seq.n - 1;
  const int nsteps = (to + STEP - 1) / STEP;

  const PackedRows kr = {p.k + int64_t(u.seq.first) * p.k_at.row + head * p.k_at.h, p.k_at.row * 2u, to};
  const PackedRows vr = {p.v + int64_t(u.seq.first) * p.v_at.row + head * p.v_at.h, p.v_at.row * 2u, to};
  auto issue = [&](int it) {
    const uint32_t at = lds + uint32_t(it & 1) * (2u * TILE * 2u);
    bwd_load_tile<D, 256, STEP>(kr.rows<D>(it * STEP), kr.pitch, 0, at, tid, w);
    bwd_load_tile<D, 256, STEP>(vr.rows<D>(it * STEP), vr.pitch, 0, at + TILE * 2u, tid, w);
  };
  issue(0);

  const int64_t at = (int64_t(u.seq.first) + token) * (p.Hk * p.G) + head * p.G + (row - token * p.G);  // row of [T * Hq]
  u32x4_t qf[KS], df[KS];
  float delta = 0.f;
  {
    const int64_t t = int64_t(u.seq.first) + token, h = head * p.G + (row - token * p.G);
    const uint16_t* q = p.q + t * p.q_row + h * p.q_head;
    const uint16_t* d = b.dout + t * b.dout_row + h * b.dout_head;
    const uint16_t* o = b.out + at * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qf[s] = *reinterpret_cast<const u32x4_t*>(q + 16 * s + 8 * g);
      df[s] = *reinterpret_cast<const u32x4_t*>(d + 16 * s + 8 * g);
      const u32x4_t of = *reinterpret_cast<const u32x4_t*>(o + 16 * s + 8 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        delta = __builtin_fmaf(widen16<BF16>(df[s][i] & 0xffffu), widen16<BF16>(of[i] & 0xffffu), delta);
        delta = __builtin_fmaf(widen16<BF16>(df[s][i] >> 16), widen16<BF16>(of[i] >> 16), delta);
      }
    }
    delta = pair_sum(delta);
    if (g == 0 && row0 + c < rows_all) b.delta[at] = delta;
  }
  const float lse2 = b.lse[at] * 1.4426950408889634f;
  const float start = CAP ? 0.f : -lse2 / p.sl2;

  f32x16_t acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16_t{};
  const uint32_t row_lane = bwd_row_lane<D>(g, c), tr_lane = bwd_tr_lane<D>(g, c, 0);
  for (int it = 0; it < nsteps; ++it) {
    wait_loads();
    __syncthreads();
    if (it + 1 < nsteps) issue(it + 1);
    const uint32_t tK = lds + uint32_t(it & 1) * (2u * TILE * 2u), tV = tK + TILE * 2u;
    const int key0 = it * STEP;
    const bool whole = key0 + STEP - 1 <= first_key && key0 + STEP <= to;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x16_t st, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        st[r] = start;
        dp[r] = -delta;
      }
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        st = mfma_32x32x16<BF16>(lds_b128_at(((tK + row_lane) ^ (32u * s)) + 32u * t * D * 2u), qf[s], st);
        dp = mfma_32x32x16<BF16>(lds_b128_at(((tV + row_lane) ^ (32u * s)) + 32u * t * D * 2u), df[s], dp);
      }
      // the row's last key, counted from the lane's first one of the tile (a score of -inf makes the weight zero)
      const int last = whole ? 0x7fffffff : (limit < to - 1 ? limit : to - 1) - key0 - 32 * t - 4 * g;
      if (!CAP && !whole) {
        static_for<16>([&](auto rc) {
          constexpr int r = decltype(rc)::value;
          if (8 * (r >> 2) + (r & 3) > last) st[r] = -INFINITY;
        });
      }
      u32x4_t pb[2];
      static_for<8>([&](auto ic) {
        constexpr int r = 2 * decltype(ic)::value;
        float ds[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if constexpr (CAP) {
            const float d = capped_d(st[r + i], p.cap_c2), th = 1.f - d;
            const float x = __builtin_amdgcn_exp2f(capped_exponent(th, b.cap_l2, -lse2)) * dp[r + i] * capped_slope(d, th);
            ds[i] = 8 * (r >> 2) + (r & 3) + i > last ? 0.f : x;
          } else {
            ds[i] = __builtin_amdgcn_exp2f(st[r + i] * p.sl2) * dp[r + i];
          }
        }
        pb[r >> 3][(r & 7) >> 1] = pack2<BF16>(ds[0], ds[1]);
      });
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          acc[dt] = mfma_32x32x16<BF16>(lds_tr_frag<D>(tK + tr_lane, 64u * dt, (32u * t + 16u * s2) * D * 2u), pb[s2], acc[dt]);
    }
  }
  __syncthreads();
  serve_store_grad<BF16, D>(acc, b.scale, reinterpret_cast<uint16_t*>(lds_raw) + w * 32 * D, lane, [&](int r) -> uint16_t* {
    const int mine = row0 + r;
    if (mine >= rows_all) return nullptr;
    const int tk = int(divide(uint32_t(mine), p.group));
    return b.dq + ((int64_t(u.seq.first) + tk) * (p.Hk * p.G) + head * p.G + (mine - tk * p.G)) * D;
  });
}

// KG groups of four waves share the rows of a tile (group i takes the steps i, i + KG, ... of its walk) and add up at the
// end.
template <bool BF16, int D, bool CAP, int KG>
__global__ void __launch_bounds__(256 * KG, 2) serve_dkdv_kernel(const ServeBwdParams b) {
  constexpr int M = 128, STEP = kDkdvStep<D>, KS = D / 16, DT = D / 32, TILE = STEP * D, CPR = D / 8;
  constexpr uint32_t SET = 2u * TILE * 2u + 2u * STEP * 4u;  // Q, dO, -LSE, -delta of a step
  const ServeParams& p = b.s;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
  const int tid = threadIdx.x & 255, lane = tid & 63, g = lane >> 5, c = lane & 31;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), kg = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 8));
  const uint32_t lds = lds_offset_of(lds_raw) + uint32_t(kg) * uint32_t(kDkdvGroupBytes<D>);
  int head, rank;
  deal_head(p, blockIdx.x, head, rank);
  if (rank >= p.units) return;
  const Unit u = find_tile<M>(p, rank, lane);
  if (!u.found) {  // keys of tokens behind the last sequence have no gradient
    if (rank < u.step0) return;
    int used = p.cu[p.B];
    used = used < 0 ? 0 : used;
    for (int64_t t = int64_t(used) + (rank - u.step0); t < p.T; t += p.units - u.step0)
      for (int i = threadIdx.x; i < D / 8; i += 256 * KG) {
        const int64_t at = (t * p.Hk + head) * D + i * 8;
        *reinterpret_cast<u32x4_t*>(b.dk + at) = u32x4_t{0u, 0u, 0u, 0u};
        *reinterpret_cast<u32x4_t*>(b.dv + at) = u32x4_t{0u, 0u, 0u, 0u};
      }
    return;
  }
  // (a causal sequence's first keys are attended by most rows: the unit that is first in the order of rows is its first)
  const int tile = p.causal ? tiles_of<M>(p, u.seq) - 1 - u.tile : u.tile;
  const int n = u.seq.n, rows_all = n * b.G, Hq = p.Hk * b.G;
  const int key0 = tile * M + 32 * w, key = key0 + c;
  const int first_row = p.causal ? tile * M * b.G : 0;           // rows that attend the tile's first key
  const int step_first = first_row / STEP, nsteps = (rows_all + STEP - 1) / STEP;
  const int whole_from = p.causal ? (key0 + 31) * b.G : 0;       // rows that attend all of the wave's keys

  constexpr bool V_IN_LDS = D == 128;
  u32x4_t kf[KS], vf[V_IN_LDS ? 1 : KS];
  const uint32_t own_v = lds_offset_of(lds_raw) + uint32_t(KG * kDkdvGroupBytes<D>) + uint32_t(w) * (32u * D * 2u);  // (of both groups)
  {
    const int64_t t = int64_t(u.seq.first) + (key < n ? key : n - 1);
    const uint16_t* k = p.k + t * p.k_at.row + head * p.k_at.h;
    const uint16_t* v = p.v + t * p.v_at.row + head * p.v_at.h;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      kf[s] = *reinterpret_cast<const u32x4_t*>(k + 16 * s + 8 * g);
      const u32x4_t x = *reinterpret_cast<const u32x4_t*>(v + 16 * s + 8 * g);
      if constexpr (V_IN_LDS) {
        *(__attribute__((address_space(3))) u32x4_t*)((own_v + bwd_row_lane<D>(g, c)) ^ (32u * s)) = x;
      } else {
        vf[s] = x;
      }
    }
  }
  // A step's rows: each lane's row is looked up (token and head of the group); rows behind the last read as zeros, and so
  // do their LSE and delta: they add nothing.
  constexpr int ROW_STRIDE = 256 / CPR, NCH = STEP / ROW_STRIDE;
  constexpr uint32_t kNowhere = 0xc0000000u, kSpan = 0xbfffffffu;  // behind the resources; a step's rows lie within 3 GiB
  auto issue = [&](int it, int set) {
    const uint32_t at = lds + uint32_t(set) * SET;
    const int r0 = it * STEP, tok0 = int(divide(uint32_t(r0), b.group));
    const int64_t t0 = int64_t(u.seq.first) + tok0;
    const i32x4_t rq = make_buffer_resource(p.q + t0 * p.q_row + int64_t(head * b.G) * p.q_head, kSpan);
    const i32x4_t rd = make_buffer_resource(b.dout + t0 * b.dout_row + int64_t(head * b.G) * b.dout_head, kSpan);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int in = tid / CPR + i * ROW_STRIDE, row = r0 + in;
      const int tk = int(divide(uint32_t(row), b.group)), h = row - tk * b.G;
      const uint32_t chunk = uint32_t((tid % CPR) ^ bwd_swizzle<D>(in)) * 16u;
      const bool live = row < rows_all;
      const uint32_t qo = live ? uint32_t((int64_t(tk - tok0) * p.q_row + h * p.q_head) * 2) + chunk : kNowhere;
      const uint32_t od = live ? uint32_t((int64_t(tk - tok0) * b.dout_row + h * b.dout_head) * 2) + chunk : kNowhere;
      buffer_to_lds_b128(rq, qo, 0, at + uint32_t(w) * 1024u + uint32_t(i) * 4096u);
      buffer_to_lds_b128(rd, od, 0, at + TILE * 2u + uint32_t(w) * 1024u + uint32_t(i) * 4096u);
    }
    if (w < 2 && lane < STEP) {  // wave 0: LSE, wave 1: delta
      const int row = r0 + lane, tk = int(divide(uint32_t(row), b.group));
      const i32x4_t rs = make_buffer_resource((w == 0 ? b.lse : b.delta) + t0 * Hq + head * b.G, kSpan);
      const uint32_t so = row < rows_all ? uint32_t(((tk - tok0) * Hq + (row - tk * b.G)) * 4) : kNowhere;
      buffer_to_lds_b32(rs, so, 0, at + 2u * TILE * 2u + uint32_t(w) * (STEP * 4u));
    }
  };
  f32x16_t dk[DT], dv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dk[dt] = dv[dt] = f32x16_t{};
  const uint32_t row_lane = bwd_row_lane<D>(g, c), tr_lane = bwd_tr_lane<D>(g, c, 0);
  const float to_start = CAP ? -1.4426950408889634f : -1.4426950408889634f / p.sl2;
  const int key_rows = p.causal ? key * b.G : 0;  // the first row that attends the lane's key
  if (step_first + kg < nsteps) issue(step_first + kg, 0);
  int set = 0;
  for (int it0 = step_first; it0 < nsteps; it0 += KG, set ^= 1) {
    const int it = it0 + kg;
    wait_loads();
    __syncthreads();
    if (it + KG < nsteps) issue(it + KG, set ^ 1);
    if (KG > 1 && it >= nsteps) break;  // (the last round of the second group: no barrier of the walk comes behind it)
    const uint32_t tQ = lds + uint32_t(set) * SET, tD = tQ + TILE * 2u, stats = tD + TILE * 2u;
    const int r0 = it * STEP;
    const bool whole = r0 >= whole_from;
#pragma unroll 1
    for (int t = 0; t < STEP / 32; ++t) {
      f32x16_t st;
      if constexpr (CAP) {
        st = f32x16_t{};
      } else {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const f32x4_t x = lds_f32x4_at(stats + uint32_t(32 * t + 8 * r4 + 4 * g) * 4u);
#pragma unroll
          for (int i = 0; i < 4; ++i) st[4 * r4 + i] = x[i] * to_start;
        }
      }
#pragma unroll
      for (int s = 0; s < KS; ++s)
        st = mfma_32x32x16<BF16>(lds_b128_at(((tQ + row_lane) ^ (32u * s)) + 32u * t * D * 2u), kf[s], st);
      const int first = key_rows - r0 - 32 * t - 4 * g;  // the step's first row that attends the key
      u32x4_t pb[2];
      static_for<4>([&](auto r4c) {
        constexpr int r4 = decltype(r4c)::value;
        f32x4_t x{};
        if constexpr (CAP) x = lds_f32x4_at(stats + uint32_t(32 * t + 8 * r4 + 4 * g) * 4u);
        float slope[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 4 * r4 + i;
          slope[i] = 1.f;
          if constexpr (CAP) {
            const float d = capped_d(st[r], p.cap_c2), th = 1.f - d;
            slope[i] = capped_slope(d, th);
            st[r] = __builtin_amdgcn_exp2f(capped_exponent(th, b.cap_l2, x[i] * to_start));
          } else {
            st[r] = __builtin_amdgcn_exp2f(st[r] * p.sl2);
          }
          if (!whole) st[r] = 8 * r4 + i < first ? 0.f : st[r];
        }
        pb[r4 >> 1][2 * (r4 & 1)] = pack2<BF16>(st[4 * r4], st[4 * r4 + 1]);
        pb[r4 >> 1][2 * (r4 & 1) + 1] = pack2<BF16>(st[4 * r4 + 2], st[4 * r4 + 3]);
        if constexpr (CAP)
#pragma unroll
          for (int i = 0; i < 4; ++i) st[4 * r4 + i] *= slope[i];  // (the products of dV have the weights packed)
      });
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          dv[dt] = mfma_32x32x16<BF16>(lds_tr_frag<D>(tD + tr_lane, 64u * dt, (32u * t + 16u * s2) * D * 2u), pb[s2], dv[dt]);
      __builtin_amdgcn_sched_barrier(0);
      f32x16_t dp;
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const f32x4_t x = lds_f32x4_at(stats + STEP * 4u + uint32_t(32 * t + 8 * r4 + 4 * g) * 4u);
#pragma unroll
        for (int i = 0; i < 4; ++i) dp[4 * r4 + i] = -x[i];
      }
#pragma unroll
      for (int s = 0; s < KS; ++s)
        dp = mfma_32x32x16<BF16>(lds_b128_at(((tD + row_lane) ^ (32u * s)) + 32u * t * D * 2u), V_IN_LDS ? lds_b128_at((own_v + row_lane) ^ (32u * s)) : vf[V_IN_LDS ? 0 : s], dp);
      static_for<8>([&](auto ic) {
        constexpr int r = 2 * decltype(ic)::value;
        pb[r >> 3][(r & 7) >> 1] = pack2<BF16>(st[r] * dp[r], st[r + 1] * dp[r + 1]);
      });
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          dk[dt] = mfma_32x32x16<BF16>(lds_tr_frag<D>(tQ + tr_lane, 64u * dt, (32u * t + 16u * s2) * D * 2u), pb[s2], dk[dt]);
    }
  }
  const auto place = [&](uint16_t* base) {
    return [=](int r) -> uint16_t* {
      return key0 + r < n ? base + ((int64_t(u.seq.first) + key0 + r) * p.Hk + head) * D : nullptr;
    };
  };
  uint16_t* stage = reinterpret_cast<uint16_t*>(lds_raw) + (4 * kg + w) * 32 * D;
  if constexpr (KG == 1) {
    __syncthreads();
    serve_store_grad<BF16, D>(dk, b.scale, stage, lane, place(b.dk));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (a wave stages both in one place)
    serve_store_grad<BF16, D>(dv, 1.f, stage, lane, place(b.dv));
    return;
  }
  // The first group gets the other's dK and stores it, the second one dV.
  constexpr int PIECES = DT * 4;  // 4-register pieces of a lane's sums
  static_assert(size_t(4) * 64 * PIECES * 16 <= 2 * kDkdvGroupBytes<D> && KG <= 2, "the tiles' place holds the sums of four waves");
  auto piece_at = [&](int piece) { return reinterpret_cast<f32x4_t*>(lds_raw) + (w * PIECES + piece) * 64 + lane; };
  auto give = [&](const f32x16_t (&x)[DT]) {
    static_for<PIECES>([&](auto pc) {
      constexpr int i = decltype(pc)::value, dt = i / 4, r = 4 * (i % 4);
      *piece_at(i) = f32x4_t{x[dt][r], x[dt][r + 1], x[dt][r + 2], x[dt][r + 3]};
    });
  };
  auto take = [&](f32x16_t (&x)[DT]) {
    static_for<PIECES>([&](auto pc) {
      constexpr int i = decltype(pc)::value, dt = i / 4, r = 4 * (i % 4);
      const f32x4_t y = *piece_at(i);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[dt][r + j] += y[j];
    });
  };
  __syncthreads();
  if (kg == 1) give(dk);
  __syncthreads();
  if (kg == 0) take(dk);
  __syncthreads();
  if (kg == 0) give(dv);
  __syncthreads();
  if (kg == 1) take(dv);
  __syncthreads();
  if (kg == 0) {
    serve_store_grad<BF16, D>(dk, b.scale, stage, lane, place(b.dk));
  } else {
    serve_store_grad<BF16, D>(dv, 1.f, stage, lane, place(b.dv));
  }
}

}  // namespace omni_attn
