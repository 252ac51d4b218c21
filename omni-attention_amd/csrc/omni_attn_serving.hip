// C ABI of the attention of packed sequences: checks, the plan of the launch, instance dispatch.
#include "../../include/omni_attn_gfx950.h"
#include "omni_attn_serving_bwd_kernel.hpp"
#include "omni_attn_serving_kernel.hpp"
#include "omni_attn_serving_plan.hpp"

#include <cmath>

namespace omni_attn {

// (beside the forward's entry points)
int device_units(int* n_xcd, int* cus);

template <bool BF16, int D>
int launch_serve(const ServeParams& p, int rows, int waves, unsigned blocks, hipStream_t stream);
template <> int launch_serve<false, 32>(const ServeParams&, int, int, unsigned, hipStream_t);
template <> int launch_serve<false, 64>(const ServeParams&, int, int, unsigned, hipStream_t);
template <> int launch_serve<false, 128>(const ServeParams&, int, int, unsigned, hipStream_t);
template <> int launch_serve<true, 32>(const ServeParams&, int, int, unsigned, hipStream_t);
template <> int launch_serve<true, 64>(const ServeParams&, int, int, unsigned, hipStream_t);
template <> int launch_serve<true, 128>(const ServeParams&, int, int, unsigned, hipStream_t);

template <bool BF16, int D>
int launch_serve_bwd(const ServeBwdParams&, unsigned, const ServeBwdParams&, unsigned, int, hipStream_t);
template <> int launch_serve_bwd<false, 32>(const ServeBwdParams&, unsigned, const ServeBwdParams&, unsigned, int, hipStream_t);
template <> int launch_serve_bwd<false, 64>(const ServeBwdParams&, unsigned, const ServeBwdParams&, unsigned, int, hipStream_t);
template <> int launch_serve_bwd<false, 128>(const ServeBwdParams&, unsigned, const ServeBwdParams&, unsigned, int, hipStream_t);
template <> int launch_serve_bwd<true, 32>(const ServeBwdParams&, unsigned, const ServeBwdParams&, unsigned, int, hipStream_t);
template <> int launch_serve_bwd<true, 64>(const ServeBwdParams&, unsigned, const ServeBwdParams&, unsigned, int, hipStream_t);
template <> int launch_serve_bwd<true, 128>(const ServeBwdParams&, unsigned, const ServeBwdParams&, unsigned, int, hipStream_t);

namespace {

bool misaligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

// Rows of 16-byte pieces; a step of 64 rows lies within 4 GiB.
int check_rows(const omni_attn_strides& at) {
  if (at.head % 8 != 0 || at.row % 8 != 0) return OMNI_ATTN_ERR_MISALIGNED;
  if (at.head < 0 || at.row < 0) return OMNI_ATTN_ERR_BAD_SHAPE;
  if (at.row > (1LL << 24)) return OMNI_ATTN_ERR_TOO_LARGE;
  return OMNI_ATTN_OK;
}

int check_sizes(int T, int B, int Hq, int Hk, int D) {
  if (D != 32 && D != 64 && D != 128) return OMNI_ATTN_ERR_UNSUPPORTED_HEAD_DIM;
  if (T <= 0 || B <= 0 || Hq <= 0 || Hk <= 0 || Hq % Hk != 0) return OMNI_ATTN_ERR_BAD_SHAPE;
  // (rows of a key head, and rows in all, are numbered with an int; a wave's rows lie within 32-bit offsets)
  if (Hq > 65536 || (long long)T * Hq > 0x3fffffffLL || (long long)B * Hk > 0x3fffffffLL) return OMNI_ATTN_ERR_TOO_LARGE;
  return OMNI_ATTN_OK;
}

// (a wave's load fills up to 16 rows, of one page)
int check_pages(int num_pages, int page_size, int max_pages) {
  if (num_pages <= 0 || max_pages <= 0 || page_size < 16 || page_size > 65536 || (page_size & (page_size - 1)) != 0)
    return OMNI_ATTN_ERR_BAD_SHAPE;
  return (long long)max_pages * page_size > 0x3fffffffLL ? OMNI_ATTN_ERR_TOO_LARGE : OMNI_ATTN_OK;
}

// Counts the units, and the places of parts, of more sequences than a wave has lanes, in one workgroup.
template <int M>
__global__ void __launch_bounds__(1024) serve_count_kernel(const ServeParams p) {
  __shared__ float steps[16];
  __shared__ int units[16], cuts[16];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  float all = 0.f;
  for (int b = tid; b < p.B; b += 1024) {
    const Sequence s = sequence_of(p, b);
    all += float(tiles_of<M>(p, s)) * float(steps_of(s.kv));
  }
  all = wave_sum(all);
  if (lane == 0) steps[w] = all;
  __syncthreads();
  all = 0.f;
  for (int i = 0; i < 16; ++i) all += steps[i];
  const int most = part_steps(p, all);
  int before = 0, cut_before = 0;
  for (int b0 = 0; b0 < p.B; b0 += 1024) {
    const Sequence s = sequence_of(p, b0 + tid);
    const int parts = parts_of(s.kv, most).n, mine = tiles_of<M>(p, s) * parts;
    const int end = wave_scan(mine), cut_end = wave_scan(parts > 1 ? mine : 0);
    if (lane == 63) {
      units[w] = end;
      cuts[w] = cut_end;
    }
    __syncthreads();
    int here = before, cut_here = cut_before;
    for (int i = 0; i < 16; ++i) {
      if (i < w) {
        here += units[i];
        cut_here += cuts[i];
      }
      before += units[i];
      cut_before += cuts[i];
    }
    if (b0 + tid < p.B) {
      p.ends[b0 + tid] = here + end;
      p.ends[p.B + 1 + b0 + tid] = cut_here + cut_end;
    }
    __syncthreads();
  }
  if (tid == 0) p.ends[p.B] = most;
}

int serve(ServeParams& p, int Hq, int D, void* workspace, size_t workspace_bytes, int dtype, float softcap, void* stream) {
  if (!(softcap >= 0.f) || std::isinf(softcap)) return OMNI_ATTN_ERR_BAD_SHAPE;
  if (dtype != OMNI_ATTN_DTYPE_F16 && dtype != OMNI_ATTN_DTYPE_BF16) return OMNI_ATTN_ERR_UNSUPPORTED_DTYPE;
  int cus = 0;
  if (const int e = device_units(&p.n_xcd, &cus)) {
    record_hip_error(e);
    return OMNI_ATTN_ERR_LAUNCH;
  }
  p.G = Hq / p.Hk;
  p.group = fast_div(uint32_t(p.G));
  p.heads = fast_div(uint32_t(p.Hk));
  const ServePlan plan = plan_serve(p.T, p.B, p.Hk, p.G, p.page_table != nullptr ? int64_t(p.max_pages) << p.page_shift : 0, cus);
  const int64_t blocks = serve_blocks(plan.units, p.Hk, p.n_xcd);
  if (blocks > 0x7fffffffLL) return OMNI_ATTN_ERR_TOO_LARGE;
  p.share = plan.share;
  p.least_steps = plan.least_steps;
  p.units = int(plan.units);
  p.places = plan.places;
  p.slots = int(plan.slots);
  if (plan.share != 0.f) {
    if (!workspace || workspace_bytes < plan.workspace_bytes(p.T, p.Hk, D)) return OMNI_ATTN_ERR_WORKSPACE;
    if (misaligned(workspace, 16)) return OMNI_ATTN_ERR_MISALIGNED;
    p.sums = static_cast<float*>(workspace);
    p.stats = p.sums + plan.slots * p.Hk * plan.rows * D;
    p.joins = reinterpret_cast<int32_t*>(p.stats + plan.slots * p.Hk * plan.rows * 2);
    p.ends = plan.counted != 0 ? p.joins + int64_t(p.T) * 4 : nullptr;
  }
  p.softcap = softcap;
  p.cap_c2 = softcap > 0.f ? float(2.0 * 1.4426950408889634 / (std::sqrt(double(D)) * double(softcap))) : 0.f;
  p.sl2 = softcap > 0.f ? float(1.4426950408889634) : float(1.4426950408889634 / std::sqrt(double(D)));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf = dtype == OMNI_ATTN_DTYPE_BF16;
  const unsigned n = unsigned(blocks);
  int e = 0;
  if (p.ends != nullptr) {
    if (plan.rows == 128) hipLaunchKernelGGL((serve_count_kernel<128>), dim3(1), dim3(1024), 0, s, p);
    else hipLaunchKernelGGL((serve_count_kernel<32>), dim3(1), dim3(1024), 0, s, p);
    e = int(hipGetLastError());
  }
  if (e == 0) switch (D) {
    case 32: e = bf ? launch_serve<true, 32>(p, plan.rows, plan.waves, n, s) : launch_serve<false, 32>(p, plan.rows, plan.waves, n, s); break;
    case 64: e = bf ? launch_serve<true, 64>(p, plan.rows, plan.waves, n, s) : launch_serve<false, 64>(p, plan.rows, plan.waves, n, s); break;
    default: e = bf ? launch_serve<true, 128>(p, plan.rows, plan.waves, n, s) : launch_serve<false, 128>(p, plan.rows, plan.waves, n, s); break;
  }
  if (e != 0) {
    record_hip_error(e);
    return OMNI_ATTN_ERR_LAUNCH;
  }
  return OMNI_ATTN_OK;
}

size_t workspace_of(int T, int B, int Hq, int Hk, int D, int64_t capacity) {
  int xcds = 0, cus = 0;
  if (check_sizes(T, B, Hq, Hk, D) != OMNI_ATTN_OK) return 0;
  if (const int e = device_units(&xcds, &cus)) {
    record_hip_error(e);
    return 0;
  }
  return plan_serve(T, B, Hk, Hq / Hk, capacity, cus).workspace_bytes(T, Hk, D);
}

}  // namespace
}  // namespace omni_attn

extern "C" size_t omni_attn_packed_workspace_bytes(int tokens, int sequences, int Hq, int Hk, int D) {
  return omni_attn::workspace_of(tokens, sequences, Hq, Hk, D, 0);
}
extern "C" size_t omni_attn_paged_workspace_bytes(int tokens, int sequences, int Hq, int Hk, int D, int page_size,
                                                  int max_pages) {
  if (omni_attn::check_pages(1, page_size, max_pages) != OMNI_ATTN_OK) return 0;
  return omni_attn::workspace_of(tokens, sequences, Hq, Hk, D, int64_t(page_size) * max_pages);
}

extern "C" int omni_attn_packed_gfx950(const void* q, const void* k, const void* v, omni_attn_strides q_at,
                                       omni_attn_strides k_at, omni_attn_strides v_at, void* o, float* lse_or_null,
                                       const int32_t* cu_seqlens, void* workspace, size_t workspace_bytes, int tokens,
                                       int sequences, int Hq, int Hk, int D, int causal, int dtype, float softcap,
                                       void* stream) {
  using namespace omni_attn;
  if (!q || !k || !v || !o || !cu_seqlens) return OMNI_ATTN_ERR_NULL_POINTER;
  if (misaligned(q, 16) || misaligned(k, 16) || misaligned(v, 16) || misaligned(o, 16) || misaligned(lse_or_null, 4) ||
      misaligned(cu_seqlens, 4))
    return OMNI_ATTN_ERR_MISALIGNED;
  if (const int rc = check_sizes(tokens, sequences, Hq, Hk, D)) return rc;
  for (const omni_attn_strides* at : {&q_at, &k_at, &v_at})
    if (const int rc = check_rows(*at)) return rc;
  ServeParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.q_row = q_at.row;
  p.q_head = q_at.head;
  p.k_at = {0, k_at.head, uint32_t(k_at.row)};
  p.v_at = {0, v_at.head, uint32_t(v_at.row)};
  p.o = static_cast<uint16_t*>(o);
  p.lse = lse_or_null;
  p.cu = cu_seqlens;
  p.T = tokens;
  p.B = sequences;
  p.Hk = Hk;
  p.causal = causal != 0;
  return serve(p, Hq, D, workspace, workspace_bytes, dtype, softcap, stream);
}

extern "C" size_t omni_attn_packed_bwd_workspace_bytes(int tokens, int Hq) {
  return tokens <= 0 || Hq <= 0 ? 0 : size_t(tokens) * size_t(Hq) * sizeof(float);
}

extern "C" int omni_attn_packed_bwd_gfx950(const void* q, const void* k, const void* v, const void* o, const void* dout,
                                           const float* lse, omni_attn_strides q_at, omni_attn_strides k_at,
                                           omni_attn_strides v_at, omni_attn_strides dout_at, void* dq, void* dk, void* dv,
                                           const int32_t* cu_seqlens, void* workspace, size_t workspace_bytes, int tokens,
                                           int sequences, int Hq, int Hk, int D, int causal, int dtype, float softcap,
                                           void* stream) {
  using namespace omni_attn;
  if (!q || !k || !v || !o || !dout || !lse || !dq || !dk || !dv || !cu_seqlens) return OMNI_ATTN_ERR_NULL_POINTER;
  for (const void* x : {q, k, v, o, dout, static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(dv)})
    if (misaligned(x, 16)) return OMNI_ATTN_ERR_MISALIGNED;
  if (misaligned(lse, 4) || misaligned(cu_seqlens, 4) || misaligned(workspace, 4)) return OMNI_ATTN_ERR_MISALIGNED;
  if (const int rc = check_sizes(tokens, sequences, Hq, Hk, D)) return rc;
  const int G = Hq / Hk;
  for (const omni_attn_strides* at : {&q_at, &k_at, &v_at, &dout_at}) {
    if (const int rc = check_rows(*at)) return rc;
    // (the rows of a step, 64 of them, lie within 3 GiB)
    if (at->head > (1LL << 30) || 66 * at->row + G * at->head > 0x5f000000LL) return OMNI_ATTN_ERR_TOO_LARGE;
  }
  if (!(softcap >= 0.f) || std::isinf(softcap)) return OMNI_ATTN_ERR_BAD_SHAPE;
  if (dtype != OMNI_ATTN_DTYPE_F16 && dtype != OMNI_ATTN_DTYPE_BF16) return OMNI_ATTN_ERR_UNSUPPORTED_DTYPE;
  if (!workspace || workspace_bytes < omni_attn_packed_bwd_workspace_bytes(tokens, Hq)) return OMNI_ATTN_ERR_WORKSPACE;
  ServeBwdParams b{};
  ServeParams& p = b.s;
  int cus = 0;
  if (const int e = device_units(&p.n_xcd, &cus)) {
    record_hip_error(e);
    return OMNI_ATTN_ERR_LAUNCH;
  }
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.q_row = q_at.row;
  p.q_head = q_at.head;
  p.k_at = {0, k_at.head, uint32_t(k_at.row)};
  p.v_at = {0, v_at.head, uint32_t(v_at.row)};
  p.o = static_cast<uint16_t*>(dq);  // (the rows that are cleared)
  p.cu = cu_seqlens;
  p.B = sequences;
  p.T = tokens;
  p.Hk = Hk;
  p.heads = fast_div(uint32_t(Hk));
  p.causal = causal != 0;
  p.softcap = softcap;
  p.cap_c2 = softcap > 0.f ? float(2.0 * 1.4426950408889634 / (std::sqrt(double(D)) * double(softcap))) : 0.f;
  p.sl2 = softcap > 0.f ? float(1.4426950408889634) : float(1.4426950408889634 / std::sqrt(double(D)));
  b.dout = static_cast<const uint16_t*>(dout);
  b.dout_row = dout_at.row;
  b.dout_head = dout_at.head;
  b.out = static_cast<const uint16_t*>(o);
  b.lse = lse;
  b.delta = static_cast<float*>(workspace);
  b.dq = static_cast<uint16_t*>(dq);
  b.dk = static_cast<uint16_t*>(dk);
  b.dv = static_cast<uint16_t*>(dv);
  b.G = G;
  b.group = fast_div(uint32_t(G));
  b.scale = float(1.0 / std::sqrt(double(D)));
  b.cap_l2 = float(1.4426950408889634 * double(softcap));
  // one unit more than there can be tiles, of rows and of keys: it clears what lies behind the last sequence
  ServeBwdParams rows = b, keys = b;
  rows.s.G = G;
  rows.s.group = b.group;
  keys.s.G = 1;
  keys.s.group = fast_div(1);
  const int64_t row_units = int64_t(tokens) * G / 128 + sequences + 1, key_units = int64_t(tokens) / 128 + sequences + 1;
  const int64_t row_blocks = serve_blocks(row_units, Hk, p.n_xcd), key_blocks = serve_blocks(key_units, Hk, p.n_xcd);
  if (row_blocks > 0x7fffffffLL || key_blocks > 0x7fffffffLL) return OMNI_ATTN_ERR_TOO_LARGE;
  rows.s.units = int(row_units);
  keys.s.units = int(key_units);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf = dtype == OMNI_ATTN_DTYPE_BF16;
  // Two groups of waves share a tile of keys where query heads share key heads (a tile then has the rows of all of them,
  // and its walk is what a launch ends with: 12 prompts of 128 - 3020 tokens, 32 / 8 heads, D=128, gradients 815 us with
  // one group, 608 with two; 2 x 4096 tokens 1185 and 980), or where there are few tiles; else one (2 x 4096 tokens, 32 /
  // 32 heads 990 us, 1034 with two; 4 x 2048, 16 / 16, D=64 182 and 201).  One, too, for many short sequences, which leave two
  // groups little to share: 32 / 8 heads, 100 prompts of 400 tokens 894 us, 1092 with two; 300 of 100 455 and 531; 2000 of 30
  // 927 and 1226 (16 of 1000, beyond the line, 607 and 617; a long prompt among short ones is what this loses by: 500 of 60 and
  // one of 4000 tokens 1312 and 1138).
  const bool many_short = tokens <= 512 * int64_t(sequences) && key_units * Hk > 8 * cus;
  const int groups = (G > 1 && !many_short) || key_units * Hk <= 2 * cus ? 2 : 1;
  const unsigned nr = unsigned(row_blocks), nk = unsigned(key_blocks);
  int e;
  switch (D) {
    case 32: e = bf ? launch_serve_bwd<true, 32>(rows, nr, keys, nk, groups, s) : launch_serve_bwd<false, 32>(rows, nr, keys, nk, groups, s); break;
    case 64: e = bf ? launch_serve_bwd<true, 64>(rows, nr, keys, nk, groups, s) : launch_serve_bwd<false, 64>(rows, nr, keys, nk, groups, s); break;
    default: e = bf ? launch_serve_bwd<true, 128>(rows, nr, keys, nk, groups, s) : launch_serve_bwd<false, 128>(rows, nr, keys, nk, groups, s); break;
  }
  if (e != 0) {
    record_hip_error(e);
    return OMNI_ATTN_ERR_LAUNCH;
  }
  return OMNI_ATTN_OK;
}

extern "C" int omni_attn_paged_gfx950(const void* q, omni_attn_strides q_at, const void* k_pages, const void* v_pages,
                                      void* o, float* lse_or_null, const int32_t* page_table, const int32_t* kv_lens,
                                      const int32_t* cu_seqlens, void* workspace, size_t workspace_bytes, int tokens,
                                      int sequences, int Hq, int Hk, int D, int num_pages, int page_size, int max_pages,
                                      int causal, int dtype, float softcap, void* stream) {
  using namespace omni_attn;
  if (!q || !k_pages || !v_pages || !o || !page_table || !kv_lens || !cu_seqlens) return OMNI_ATTN_ERR_NULL_POINTER;
  if (misaligned(q, 16) || misaligned(k_pages, 16) || misaligned(v_pages, 16) || misaligned(o, 16) ||
      misaligned(lse_or_null, 4) || misaligned(page_table, 4) || misaligned(kv_lens, 4) || misaligned(cu_seqlens, 4))
    return OMNI_ATTN_ERR_MISALIGNED;
  if (const int rc = check_sizes(tokens, sequences, Hq, Hk, D)) return rc;
  if (const int rc = check_rows(q_at)) return rc;
  if (const int rc = check_pages(num_pages, page_size, max_pages)) return rc;
  ServeParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k_pages);
  p.v = static_cast<const uint16_t*>(v_pages);
  p.q_row = q_at.row;
  p.q_head = q_at.head;
  p.o = static_cast<uint16_t*>(o);
  p.lse = lse_or_null;
  p.cu = cu_seqlens;
  p.kv_lens = kv_lens;
  p.page_table = page_table;
  p.num_pages = num_pages;
  p.max_pages = max_pages;
  p.page_shift = __builtin_ctz(unsigned(page_size));
  p.T = tokens;
  p.B = sequences;
  p.Hk = Hk;
  p.causal = causal != 0;
  return serve(p, Hq, D, workspace, workspace_bytes, dtype, softcap, stream);
}
