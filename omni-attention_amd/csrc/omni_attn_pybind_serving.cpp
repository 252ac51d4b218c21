// Python module `omni_attn`, second part: norm and rotation of query and key heads (differentiable), the paged
// cache's append, and the attention of packed sequences over their own keys or a paged cache.  Host-only C++ over
// include/omni_attn_gfx950.h; the reference has no counterpart of these operators.
#include <torch/extension.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <stdexcept>
#include <string>
#include <vector>

#include "omni_attn_gfx950.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

[[noreturn]] void refuse(const std::string& what) { throw pybind11::value_error(what); }
void require(bool ok, const char* what) {
  if (!ok) refuse(what);
}
[[noreturn]] void fail(int rc) {
  std::string msg = std::string("omni_attn: ") + omni_attn_status_string(rc);
  if (rc == OMNI_ATTN_ERR_LAUNCH) msg += " (hipError " + std::to_string(omni_attn_last_hip_error()) + ")";
  throw std::runtime_error(msg);
}
int dtype_of(const Tensor& t) { return t.scalar_type() == torch::kBFloat16 ? OMNI_ATTN_DTYPE_BF16 : OMNI_ATTN_DTYPE_F16; }
void* stream_of(const Tensor& t) {
  return static_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

void check_operand(const Tensor& t, const char* name, const Tensor& like) {
  const std::string n(name);
  if (!t.is_cuda()) refuse(n + " must be a GPU tensor");
  if (t.device() != like.device()) refuse(n + " must be on the device of the other operands");
  if (t.scalar_type() != torch::kHalf && t.scalar_type() != torch::kBFloat16)
    refuse(n + " must be torch.float16 or torch.bfloat16");
  if (t.scalar_type() != like.scalar_type()) refuse(n + " must have the dtype of the other operands");
}
void check_int32(const Tensor& t, const char* name, const Tensor& like, int64_t dims) {
  const std::string n(name);
  if (t.scalar_type() != torch::kInt32) refuse(n + " must be torch.int32");
  if (t.device() != like.device()) refuse(n + " must be on the device of the operands");
  if (t.dim() != dims) refuse(n + " must have " + std::to_string(dims) + " dimension" + (dims == 1 ? "" : "s"));
}
// These operators keep nothing for a backward pass: a gradient that would be missing is refused.
void check_no_grad(std::initializer_list<Tensor> tensors, const char* op) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor& t : tensors)
    if (t.defined() && t.requires_grad())
      refuse(std::string(op) + " is not differentiable: call it under torch.no_grad()");
}

// A tangent of forward-mode differentiation would be dropped without a word, also under torch.no_grad().
void check_no_tangent(std::initializer_list<Tensor> tensors, const char* op) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor& t : tensors)
    if (t.defined() && t._fw_grad(/*level=*/0).defined())
      refuse(std::string(op) + " has no forward-mode derivative: its operands must not have tangents");
}

// Rows that the kernels read in place: whole pieces of `piece` elements, up to 2^24 apart ([B, H, S, D]: 2^31).  Others are
// copied.
Tensor in_rows(const Tensor& t, int64_t piece) {
  bool ok = t.stride(-1) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & uintptr_t(2 * piece - 1)) == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && t.stride(i) >= 0 && t.stride(i) % piece == 0;
  ok = ok && (t.dim() == 3 ? t.stride(0) <= (1 << 24) && t.stride(1) <= (1 << 30) : t.stride(2) <= 0x7fffffff);
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
// ... for the gradients of packed sequences, too: a step's rows, of every head, within 3 GiB.
Tensor in_near_rows(const Tensor& t) {
  const Tensor r = in_rows(t, 8);
  return 66 * r.stride(0) + r.size(1) * r.stride(1) <= 0x5f000000 ? r : r.clone(at::MemoryFormat::Contiguous);
}
Tensor aligned(const Tensor& t) {  // contiguous and on a 16-byte boundary
  if (t.is_contiguous() && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}
// [T, H, D] or [B, H, S, D] as batch, head and row strides.
omni_attn_strides strides_of(const Tensor& t) {
  if (t.dim() == 3) return {0, t.stride(1), t.stride(0)};
  return {t.stride(0), t.stride(1), t.stride(2)};
}
// A result in the memory order of its operand (a projection's [B, S, H, D] seen as [B, H, S, D] stays that).
Tensor result_like(const Tensor& t) {
  if (t.dim() == 4 && t.stride(1) < t.stride(2)) {
    const int64_t B = t.size(0), H = t.size(1), S = t.size(2), D = t.size(3);
    return at::empty_strided({B, H, S, D}, {S * H * D, D, H * D, 1}, t.options());
  }
  return at::empty(t.sizes(), t.options());
}

// ---- norm and rotation ------------------------------------------------------------------------------

struct Rotation {
  Tensor positions, table, wq, wk;  // weights may be undefined
  double eps = 0;
  bool interleaved = false;
  int64_t pos_b = 0;  // distance of two batch elements' positions
};

void check_weight(const Tensor& w, const char* name, const Tensor& like, int64_t D) {
  if (!w.defined()) return;
  const std::string n(name);
  if (w.device() != like.device()) refuse(n + " must be on the device of the operands");
  if (w.dim() != 1 || w.size(0) != D) refuse(n + " must have one weight per dimension of a head");
  if (w.scalar_type() != like.scalar_type() && w.scalar_type() != torch::kFloat32)
    refuse(n + " must have the dtype of the operands or torch.float32");
}
void check_rotation(Rotation& r, const Tensor& q, int64_t D) {
  check_weight(r.wq, "query_norm", q, D);
  check_weight(r.wk, "key_norm", q, D);
  if (r.wq.defined() && r.wk.defined() && r.wq.scalar_type() != r.wk.scalar_type())
    refuse("query_norm and key_norm must have one dtype");
  if (!(r.eps >= 0) || std::isinf(r.eps)) refuse("eps must be a finite number that is not negative");
  if (r.table.defined()) {
    if (r.table.scalar_type() != torch::kFloat32 || r.table.dim() != 2 || r.table.device() != q.device())
      refuse("table must be a torch.float32 tensor [positions, rotary_dim] on the device of the operands");
    if (r.table.size(0) < 1 || r.table.size(0) > 0x7fffffff) refuse("table must have at least one position");
    const int64_t rot = r.table.size(1);
    if (rot < 8 || rot > D || rot % 8 != 0)
      refuse("Unsupported rotary_dim=" + std::to_string(rot) + ". Supported values: multiples of 8 up to head_dim.");
    r.table = aligned(r.table);
  }
  if (r.wq.defined()) r.wq = aligned(r.wq);
  if (r.wk.defined()) r.wk = aligned(r.wk);
}
// Learned frequencies have no gradient here: refused, where one would be missing.
void check_table_grad(const Tensor& table) {
  if (at::GradMode::is_enabled() && table.defined() && table.requires_grad())
    refuse("table must not require a gradient: the operators have none for it");
}
void check_head_dim(int64_t D) {
  if (D < 8 || D > 256 || D % 8 != 0)
    refuse("Unsupported head_dim=" + std::to_string(D) + ". Supported values: multiples of 8 up to 256.");
}
void check_positions(const Tensor& p, const Tensor& like) {
  if (p.scalar_type() != torch::kInt32 && p.scalar_type() != torch::kInt64) refuse("positions must be torch.int32 or torch.int64");
  if (p.device() != like.device()) refuse("positions must be on the device of the operands");
}
bool weights_f32(const Rotation& r) {
  return (r.wq.defined() && r.wq.scalar_type() == torch::kFloat32) || (r.wk.defined() && r.wk.scalar_type() == torch::kFloat32);
}
const void* ptr_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

std::pair<Tensor, Tensor> rotate(const Tensor& q, const Tensor& k, const Rotation& r) {
  Tensor qo = result_like(q), ko = result_like(k);
  const bool flat = q.dim() == 3;
  const int64_t B = flat ? 1 : q.size(0), S = flat ? q.size(0) : q.size(2);
  if (B == 0 || S == 0) return {qo, ko};
  const int rc = omni_attn_qk_rotary_gfx950(
      q.data_ptr(), k.data_ptr(), strides_of(q), strides_of(k), qo.data_ptr(), ko.data_ptr(), strides_of(qo), strides_of(ko),
      r.table.data_ptr<float>(), r.positions.data_ptr(), r.pos_b, r.positions.scalar_type() == torch::kInt64,
      ptr_or_null(r.wq), ptr_or_null(r.wk), weights_f32(r), int(B), int(S), int(q.size(1)), int(k.size(1)), int(q.size(-1)),
      int(r.table.size(1)), int(r.table.size(0)), float(r.eps), r.interleaved, dtype_of(q), stream_of(q));
  if (rc != OMNI_ATTN_OK) fail(rc);
  return {qo, ko};
}

class RotaryFunction : public torch::autograd::Function<RotaryFunction> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, Tensor q, Tensor k, OptTensor query_norm,
                                                OptTensor key_norm, const Rotation& given) {
    Rotation r = given;
    const Tensor wq = query_norm.value_or(Tensor()), wk = key_norm.value_or(Tensor());
    r.wq = wq;
    r.wk = wk;
    q = in_rows(q, 4);
    k = in_rows(k, 4);
    auto out = rotate(q, k, r);
    // (a rotation alone needs no inputs for its gradient)
    ctx->save_for_backward({wq.defined() ? q : Tensor(), wk.defined() ? k : Tensor(), r.positions, r.table, wq, wk});
    ctx->saved_data["eps"] = r.eps;
    ctx->saved_data["how"] = r.pos_b * 8 + int64_t(r.interleaved) * 4 + int64_t(wq.defined() && wq.requires_grad()) * 2 +
                             int64_t(wk.defined() && wk.requires_grad());
    return {out.first, out.second};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    if (at::GradMode::is_enabled())
      throw std::runtime_error("omni_qk_rotary: gradients of its gradients are not implemented");
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1];
    Rotation r;
    r.positions = saved[2];
    r.table = saved[3];
    r.wq = saved[4];
    r.wk = saved[5];
    r.eps = ctx->saved_data["eps"].toDouble();
    const int64_t how = ctx->saved_data["how"].toInt();
    r.interleaved = (how & 4) != 0;
    r.pos_b = how >> 3;
    c10::DeviceGuard guard(r.table.device());
    // (the gradient of an output that nothing was computed from comes as zeros)
    const Tensor dqo = in_rows(grads[0], 4), dko = in_rows(grads[1], 4);
    Tensor dq = result_like(dqo), dk = result_like(dko);
    const bool want_wq = (how & 2) != 0, want_wk = (how & 1) != 0;
    Tensor dwq, dwk, workspace;
    const bool flat = dqo.dim() == 3;
    const int64_t B = flat ? 1 : dqo.size(0), S = flat ? dqo.size(0) : dqo.size(2), D = dqo.size(-1);
    if (want_wq) dwq = B * S == 0 ? torch::zeros_like(r.wq) : torch::empty_like(r.wq);
    if (want_wk) dwk = B * S == 0 ? torch::zeros_like(r.wk) : torch::empty_like(r.wk);
    if (B * S != 0) {
      const size_t bytes = want_wq || want_wk ? omni_attn_qk_rotary_bwd_workspace_bytes(int(B), int(S), int(D)) : 0;
      if (bytes) workspace = torch::empty({int64_t(bytes / 4)}, r.table.options());
      const omni_attn_strides none{0, 0, 0};
      const int rc = omni_attn_qk_rotary_bwd_gfx950(
          dqo.data_ptr(), dko.data_ptr(), ptr_or_null(q), ptr_or_null(k), strides_of(dqo), strides_of(dko),
          q.defined() ? strides_of(q) : none, k.defined() ? strides_of(k) : none, dq.data_ptr(), dk.data_ptr(), strides_of(dq),
          strides_of(dk), want_wq ? dwq.data_ptr() : nullptr, want_wk ? dwk.data_ptr() : nullptr, r.table.data_ptr<float>(),
          r.positions.data_ptr(), r.pos_b, r.positions.scalar_type() == torch::kInt64, ptr_or_null(r.wq), ptr_or_null(r.wk),
          weights_f32(r), bytes ? workspace.data_ptr() : nullptr, bytes, int(B), int(S), int(dqo.size(1)), int(dko.size(1)), int(D),
          int(r.table.size(1)), int(r.table.size(0)), float(r.eps), r.interleaved, dtype_of(dqo), stream_of(dqo));
      if (rc != OMNI_ATTN_OK) fail(rc);
    }
    return {dq, dk, dwq, dwk, Tensor()};
  }
};

pybind11::tuple omni_attn_qk_rotary(Tensor q, Tensor k, Tensor positions, Tensor table, OptTensor wq, OptTensor wk, double eps,
                                    bool interleaved) {
  check_no_tangent({q, k, table, wq.value_or(Tensor()), wk.value_or(Tensor())}, "omni_qk_rotary");
  check_table_grad(table);
  check_operand(q, "query", q);
  check_operand(k, "key", q);
  require((q.dim() == 3 || q.dim() == 4) && k.dim() == q.dim(), "query and key must be [tokens, heads, head_dim] or [B, H, S, D]");
  const bool flat = q.dim() == 3;
  const int64_t S = flat ? q.size(0) : q.size(2), D = q.size(-1);
  check_head_dim(D);
  require(k.size(-1) == D && (flat ? k.size(0) == S : (k.size(0) == q.size(0) && k.size(2) == S)),
          "query and key must have the same tokens and head_dim");
  require(q.size(1) >= 1 && k.size(1) >= 1, "query and key must have heads");
  require(q.size(1) <= 65536 && k.size(1) <= 65536 && S <= 0x7fffffff && (flat || q.size(0) <= 0x7fffffff),
          "query or key is too large");
  check_positions(positions, q);
  Rotation r;
  const bool per_batch = !flat && positions.dim() == 2;
  require(per_batch ? positions.size(0) == q.size(0) && positions.size(1) == S : positions.dim() == 1 && positions.size(0) == S,
          "positions must have one entry per token: [S], or [B, S] for [B, H, S, D] operands");
  r.positions = positions.contiguous();
  r.pos_b = per_batch ? S : 0;
  r.table = table;
  r.eps = eps;
  r.interleaved = interleaved;
  if (wq) r.wq = *wq;
  if (wk) r.wk = *wk;
  c10::DeviceGuard guard(q.device());
  check_rotation(r, q, D);
  const auto if_defined = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
  const OptTensor query_norm = if_defined(r.wq), key_norm = if_defined(r.wk);
  auto out = RotaryFunction::apply(q, k, query_norm, key_norm, r);
  return pybind11::make_tuple(std::move(out[0]), std::move(out[1]));
}

// ---- the cache ---------------------------------------------------------------------------------------

struct Pages {
  int64_t num, Hk, size, D;
};
Pages check_pages(const Tensor& kp, const Tensor& vp, const Tensor& like) {
  check_operand(kp, "key_pages", like);
  check_operand(vp, "value_pages", like);
  require(kp.dim() == 4 && kp.sizes() == vp.sizes(), "key_pages and value_pages must be [num_pages, kv_heads, page_size, head_dim]");
  require(kp.is_contiguous() && vp.is_contiguous(), "key_pages and value_pages must be contiguous");
  require((reinterpret_cast<uintptr_t>(kp.data_ptr()) & 15) == 0 && (reinterpret_cast<uintptr_t>(vp.data_ptr()) & 15) == 0,
          "key_pages and value_pages must start on a 16-byte boundary");
  const Pages p{kp.size(0), kp.size(1), kp.size(2), kp.size(3)};
  require(p.num >= 1 && p.num <= 0x7fffffff && p.Hk >= 1, "the cache must have pages and heads");
  if (p.size < 16 || p.size > 65536 || (p.size & (p.size - 1)) != 0)
    refuse("Unsupported page_size=" + std::to_string(p.size) + ". Supported values: powers of two from 16 to 65536.");
  return p;
}
// page_table [B, max_pages], kv_lens [B], cu_seqlens [B + 1].
int64_t check_batch(Tensor& table, Tensor& lens, Tensor& cu, const Tensor& like, const Pages& pages) {
  check_int32(table, "page_table", like, 2);
  check_int32(lens, "kv_lens", like, 1);
  check_int32(cu, "cu_seqlens", like, 1);
  const int64_t B = lens.size(0);
  require(cu.size(0) == B + 1, "cu_seqlens must have one entry more than kv_lens");
  require(table.size(0) == B, "page_table must have a row per sequence");
  require(B == 0 || table.size(1) >= 1, "page_table must have columns");
  require(table.size(1) * pages.size <= 0x3fffffff, "page_table has room for too many keys");
  table = table.contiguous();
  lens = lens.contiguous();
  cu = cu.contiguous();
  return B;
}

pybind11::object omni_attn_cache_append(Tensor k, Tensor v, Tensor k_pages, Tensor v_pages, Tensor page_table, Tensor kv_lens,
                                        Tensor cu, OptTensor table, OptTensor positions, OptTensor query, OptTensor wq,
                                        OptTensor wk, double eps, bool interleaved) {
  check_no_tangent({k, v, k_pages, v_pages, table.value_or(Tensor()), query.value_or(Tensor()), wq.value_or(Tensor()),
                    wk.value_or(Tensor())}, "omni_cache_append");
  check_table_grad(table.value_or(Tensor()));
  check_operand(k, "key", k);
  check_operand(v, "value", k);
  require(k.dim() == 3 && k.sizes() == v.sizes(), "key and value must be [tokens, kv_heads, head_dim]");
  const Pages pages = check_pages(k_pages, v_pages, k);
  const int64_t T = k.size(0), D = k.size(2);
  check_head_dim(D);
  require(pages.Hk == k.size(1) && pages.D == D, "key_pages must have the heads and head_dim of key");
  {
    const char *a = static_cast<const char*>(k_pages.data_ptr()), *b = static_cast<const char*>(v_pages.data_ptr());
    require((a > b ? a - b : b - a) >= int64_t(k_pages.nbytes()), "key_pages and value_pages must not overlap");
  }
  require(k.size(1) <= 65536 && T <= 0x7fffffff, "key is too large");
  c10::DeviceGuard guard(k.device());
  const int64_t B = check_batch(page_table, kv_lens, cu, k, pages);
  Rotation r;
  r.eps = eps;
  r.interleaved = interleaved;
  if (table) r.table = *table;
  if (wq) r.wq = *wq;
  if (wk) r.wk = *wk;
  require(!r.wq.defined() || query, "query_norm without query");
  require(!positions || table, "positions without table");
  check_rotation(r, k, D);
  Tensor q;
  if (query) {
    q = *query;
    check_operand(q, "query", k);
    require(q.dim() == 3 && q.size(0) == T && q.size(2) == D && q.size(1) >= 1 && q.size(1) <= 65536,
            "query must be [tokens, heads, head_dim] with the tokens and head_dim of key");
  }
  if (positions) {
    check_positions(*positions, k);
    require(positions->dim() == 1 && positions->size(0) == T, "positions must have one entry per token");
    r.positions = positions->contiguous();
  }
  check_no_grad({k, v, q, r.wq, r.wk, k_pages, v_pages}, "omni_cache_append");
  at::NoGradGuard no_grad;
  Tensor q_out;
  if (q.defined()) q_out = torch::empty(q.sizes(), q.options());
  if (T != 0 && B != 0) {
    k = in_rows(k, 4);
    v = in_rows(v, 4);
    if (q.defined()) q = in_rows(q, 4);
    // (what autograd has saved of the pages is no longer theirs; refuses what may not be written)
    k_pages.unsafeGetTensorImpl()->bump_version();
    v_pages.unsafeGetTensorImpl()->bump_version();
    const omni_attn_strides none{0, 0, 0};
    const bool turns = r.table.defined();
    const int rc = omni_attn_cache_append_gfx950(
        ptr_or_null(q), k.data_ptr(), v.data_ptr(), q.defined() ? strides_of(q) : none, strides_of(k), strides_of(v),
        q.defined() ? q_out.data_ptr() : nullptr, q.defined() ? strides_of(q_out) : none, k_pages.data_ptr(), v_pages.data_ptr(),
        page_table.data_ptr<int32_t>(), kv_lens.data_ptr<int32_t>(), cu.data_ptr<int32_t>(),
        turns ? r.table.data_ptr<float>() : nullptr, ptr_or_null(r.positions),
        r.positions.defined() && r.positions.scalar_type() == torch::kInt64, ptr_or_null(r.wq), ptr_or_null(r.wk), weights_f32(r),
        int(T), int(B), q.defined() ? int(q.size(1)) : 0, int(k.size(1)), int(D), int(pages.num), int(pages.size),
        int(page_table.size(1)), turns ? int(r.table.size(1)) : 0, turns ? int(r.table.size(0)) : 0, float(r.eps), r.interleaved,
        dtype_of(k), stream_of(k));
    if (rc != OMNI_ATTN_OK) fail(rc);
  } else if (q_out.defined()) {
    q_out.zero_();
  }
  if (!q_out.defined()) return pybind11::none();
  return pybind11::cast(std::move(q_out));
}

// ---- attention of packed sequences -------------------------------------------------------------------

void check_heads(const Tensor& q, int64_t Hk, int64_t D) {
  if (D != 32 && D != 64 && D != 128)
    refuse("Unsupported head_dim=" + std::to_string(D) + ". Supported values: 32, 64, 128.");
  require(q.size(1) >= 1 && Hk >= 1 && q.size(1) % Hk == 0, "the number of query heads must be a multiple of the key heads'");
  require(q.size(1) <= 65536 && q.size(0) * q.size(1) <= 0x3fffffff, "query has too many rows");
}
void check_softcap(double softcap) {
  if (!(softcap >= 0) || std::isinf(softcap)) refuse("softcap must be 0 (off) or positive and finite");
}
pybind11::object result(Tensor out, Tensor lse, bool want_lse) {
  if (want_lse) return pybind11::make_tuple(std::move(out), std::move(lse));
  return pybind11::cast(std::move(out));
}

struct Packed {
  Tensor cu;
  bool causal = true;
  double softcap = 0;
};
// q, k and v become the tensors the kernel has read (copies where it could not read them in place).
Tensor attend_packed(Tensor& q, Tensor& k, Tensor& v, const Packed& m, Tensor* lse) {
  const int64_t T = q.size(0), B = m.cu.size(0) - 1, Hq = q.size(1), Hk = k.size(1), D = q.size(2);
  const auto f32 = q.options().dtype(torch::kFloat32);
  if (T == 0 || B == 0) {
    if (lse) *lse = torch::full({T, Hq}, -std::numeric_limits<float>::infinity(), f32);
    return torch::zeros({T, Hq, D}, q.options());
  }
  q = in_rows(q, 8);
  k = in_rows(k, 8);
  v = in_rows(v, 8);
  Tensor out = torch::empty({T, Hq, D}, q.options()), workspace;
  if (lse) *lse = torch::empty({T, Hq}, f32);
  const size_t bytes = omni_attn_packed_workspace_bytes(int(T), int(B), int(Hq), int(Hk), int(D));
  if (bytes) workspace = torch::empty({int64_t((bytes + 3) / 4)}, f32);
  const int rc = omni_attn_packed_gfx950(q.data_ptr(), k.data_ptr(), v.data_ptr(), strides_of(q), strides_of(k), strides_of(v),
                                         out.data_ptr(), lse ? lse->data_ptr<float>() : nullptr, m.cu.data_ptr<int32_t>(),
                                         bytes ? workspace.data_ptr() : nullptr, bytes, int(T), int(B), int(Hq), int(Hk), int(D),
                                         m.causal, dtype_of(q), float(m.softcap), stream_of(q));
  if (rc != OMNI_ATTN_OK) fail(rc);
  return out;
}

class PackedFunction : public torch::autograd::Function<PackedFunction> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, Tensor q, Tensor k, Tensor v, const Packed& m) {
    Tensor lse;
    q = in_near_rows(q);
    k = in_near_rows(k);
    v = in_near_rows(v);
    Tensor out = attend_packed(q, k, v, m, &lse);
    ctx->save_for_backward({q, k, v, out, lse, m.cu});
    ctx->saved_data["causal"] = m.causal;
    ctx->saved_data["softcap"] = m.softcap;
    ctx->mark_non_differentiable({lse});
    return {out, lse};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    if (at::GradMode::is_enabled())
      throw std::runtime_error("omni_attention_packed: gradients of its gradients are not implemented");
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3], &lse = saved[4], &cu = saved[5];
    const int64_t T = q.size(0), B = cu.size(0) - 1, Hq = q.size(1), Hk = k.size(1), D = q.size(2);
    c10::DeviceGuard guard(q.device());
    if (T == 0 || B == 0) return {torch::zeros_like(q), torch::zeros_like(k), torch::zeros_like(v), Tensor()};
    const Tensor dout = in_near_rows(grads[0]);
    Tensor dq = torch::empty({T, Hq, D}, q.options()), dk = torch::empty({T, Hk, D}, q.options()), dv = torch::empty({T, Hk, D}, q.options());
    const size_t bytes = omni_attn_packed_bwd_workspace_bytes(int(T), int(Hq));
    Tensor workspace = torch::empty({int64_t(bytes / 4)}, lse.options());
    const int rc = omni_attn_packed_bwd_gfx950(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(), lse.data_ptr<float>(), strides_of(q), strides_of(k),
        strides_of(v), strides_of(dout), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), cu.data_ptr<int32_t>(), workspace.data_ptr(),
        bytes, int(T), int(B), int(Hq), int(Hk), int(D), ctx->saved_data["causal"].toBool(), dtype_of(q),
        float(ctx->saved_data["softcap"].toDouble()), stream_of(q));
    if (rc != OMNI_ATTN_OK) fail(rc);
    return {dq, dk, dv, Tensor()};
  }
};

pybind11::object omni_attn_packed(Tensor q, Tensor k, Tensor v, Tensor cu, bool causal, double softcap, bool want_lse) {
  check_no_tangent({q, k, v}, "omni_attention_packed");
  check_operand(q, "query", q);
  check_operand(k, "key", q);
  check_operand(v, "value", q);
  require(q.dim() == 3 && k.dim() == 3 && k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(2) == q.size(2),
          "query must be [tokens, heads, head_dim], key and value [tokens, kv_heads, head_dim]");
  check_heads(q, k.size(1), q.size(2));
  check_int32(cu, "cu_seqlens", q, 1);
  require(cu.size(0) >= 1, "cu_seqlens must have one entry more than there are sequences");
  check_softcap(softcap);
  require((cu.size(0) - 1) * k.size(1) <= 0x3fffffff, "too many sequences");
  c10::DeviceGuard guard(q.device());
  const Packed m{cu.contiguous(), causal, softcap};
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad())) {
    auto out = PackedFunction::apply(q, k, v, m);
    return result(std::move(out[0]), std::move(out[1]), want_lse);
  }
  at::NoGradGuard no_grad;
  Tensor lse;
  Tensor out = attend_packed(q, k, v, m, want_lse ? &lse : nullptr);
  return result(std::move(out), std::move(lse), want_lse);
}

pybind11::object omni_attn_paged(Tensor q, Tensor k_pages, Tensor v_pages, Tensor page_table, Tensor kv_lens, Tensor cu,
                                 bool causal, double softcap, bool want_lse) {
  check_no_tangent({q, k_pages, v_pages}, "omni_attention_paged");
  check_operand(q, "query", q);
  require(q.dim() == 3, "query must be [tokens, heads, head_dim]");
  const Pages pages = check_pages(k_pages, v_pages, q);
  require(pages.D == q.size(2), "key_pages must have the head_dim of query");
  check_heads(q, pages.Hk, q.size(2));
  check_softcap(softcap);
  check_no_grad({q, k_pages, v_pages}, "omni_attention_paged");
  at::NoGradGuard no_grad;
  c10::DeviceGuard guard(q.device());
  const int64_t B = check_batch(page_table, kv_lens, cu, q, pages);
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
  require(B * pages.Hk <= 0x3fffffff, "too many sequences");
  const bool some = T != 0 && B != 0;
  Tensor out = some ? torch::empty({T, Hq, D}, q.options()) : torch::zeros({T, Hq, D}, q.options()), lse;
  if (want_lse) {
    const auto f32 = q.options().dtype(torch::kFloat32);
    lse = some ? torch::empty({T, Hq}, f32) : torch::full({T, Hq}, -std::numeric_limits<float>::infinity(), f32);
  }
  if (some) {
    q = in_rows(q, 8);
    const size_t bytes = omni_attn_paged_workspace_bytes(int(T), int(B), int(Hq), int(pages.Hk), int(D), int(pages.size),
                                                         int(page_table.size(1)));
    Tensor workspace;
    if (bytes) workspace = torch::empty({int64_t((bytes + 3) / 4)}, q.options().dtype(torch::kFloat32));
    const int rc = omni_attn_paged_gfx950(q.data_ptr(), strides_of(q), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(),
                                          want_lse ? lse.data_ptr<float>() : nullptr, page_table.data_ptr<int32_t>(),
                                          kv_lens.data_ptr<int32_t>(), cu.data_ptr<int32_t>(),
                                          bytes ? workspace.data_ptr() : nullptr, bytes, int(T), int(B), int(Hq), int(pages.Hk),
                                          int(D), int(pages.num), int(pages.size), int(page_table.size(1)), causal, dtype_of(q),
                                          float(softcap), stream_of(q));
    if (rc != OMNI_ATTN_OK) fail(rc);
  }
  return result(std::move(out), std::move(lse), want_lse);
}

}  // namespace

void bind_serving(pybind11::module& m) {
  m.def("omni_attn_qk_rotary", &omni_attn_qk_rotary, "omni_attn_qk_rotary (norm and rotation of query and key heads)");
  m.def("omni_attn_cache_append", &omni_attn_cache_append, "omni_attn_cache_append (new tokens into a paged cache)");
  m.def("omni_attn_packed", &omni_attn_packed, "omni_attn_packed (attention of packed sequences)");
  m.def("omni_attn_paged", &omni_attn_paged, "omni_attn_paged (attention of new tokens over a paged cache)");
}
