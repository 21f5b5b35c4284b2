// PyTorch operator registration of the DSA kernels: torch.ops.dsa.*.
//
// The pattern of examples/torch_tl_ascend/src/_inner.cpp:17-68 (a wrapper that
// allocates outputs and workspaces with ATen, fetches the current stream and
// calls the C entry point; TORCH_LIBRARY schemas; device and Meta
// implementations), for a HIP device: the device implementations call the C
// ABI of include/dsa_mi355x.h on the current HIP stream; the Meta
// implementations only compute output shapes, so the ops trace under
// torch.compile / FakeTensor.  No implementation synchronises with the host or
// allocates outside ATen's caching allocator, so the calls can be captured in a
// HIP graph.  Sizes that the Python wrappers read from device tensors (the
// longest paged key length, the compressed-row bound of V4 "hca") are explicit
// arguments here.
//
// Every tensor argument, optional ones included, is checked before anything is
// launched: on the main tensor's device, of the expected element count / shape,
// and made contiguous in the dtype the kernel reads (a host tensor or a short
// buffer raises here instead of reaching a kernel).
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include "../../include/dsa_mi355x.h"

namespace {

void* ptr(const at::Tensor& t) { return t.data_ptr(); }
template <typename T>
T* ptr_or_null(const c10::optional<at::Tensor>& t) {
  return t.has_value() ? static_cast<T*>(t->data_ptr()) : nullptr;
}

void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == 0, "dsa.", what, ": ", dsa_last_error_message(), " (hipError ", rc, ")");
}

int kind_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat8_e4m3fn: return DSA_KIND_FP8_E4M3;
    case at::kBFloat16: return DSA_KIND_BF16;
    case at::kHalf: return DSA_KIND_FP16;
    case at::kFloat: return DSA_KIND_FP32;
    case at::kChar: return DSA_KIND_INT8;
    default: TORCH_CHECK(false, "dsa: unsupported dtype ", t.scalar_type());
  }
  return -1;
}

void require(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "dsa: ", name, " must be on a HIP device");
  TORCH_CHECK(t.is_contiguous(), "dsa: ", name, " must be contiguous");
}

// A tensor a kernel reads lives on the main tensor's device: a host tensor (the
// torch_npu convention for actual_seq_lengths) or one on another GPU would hand
// the kernel an address it cannot read.
void require_on(const at::Tensor& t, const at::Tensor& main, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == main.device(), "dsa: ", name, " must be on ", main.device(), " (got ",
              t.device(), ")");
}

void require_numel(const at::Tensor& t, int64_t n, const char* name) {
  TORCH_CHECK(t.numel() == n, "dsa: ", name, " must have ", n, " elements (got ", t.numel(), ")");
}

bool is_int(const at::Tensor& t) {
  return at::isIntegralType(t.scalar_type(), /*includeBool=*/false);
}

// An int32 argument: on main's device, integral, `n` elements (n < 0: any), made contiguous int32.
at::Tensor aux_i32(const at::Tensor& t, const at::Tensor& main, int64_t n, const char* name) {
  require_on(t, main, name);
  TORCH_CHECK(is_int(t), "dsa: ", name, " must be an integer tensor (got ", t.scalar_type(), ")");
  if (n >= 0) require_numel(t, n, name);
  return t.to(at::kInt).contiguous();
}

c10::optional<at::Tensor> aux_i32(const c10::optional<at::Tensor>& t, const at::Tensor& main, int64_t n,
                                  const char* name) {
  if (!t.has_value()) return t;
  return aux_i32(*t, main, n, name);
}

// Integers whose values past 32 bits lie at the ends of that range: cast as they are they would wrap into it.
at::Tensor saturated_i32(const at::Tensor& t) {
  const at::ScalarType st = t.scalar_type();
  if (st != at::kLong && st != at::kUInt32 && st != at::kUInt64) return t;
  at::Tensor wide = t.to(at::kLong);
  if (st == at::kUInt64) wide = wide.masked_fill(wide < 0, 0x7fffffff);  // values past 63 bits have come out negative
  return wide.clamp(-0x80000000LL, 0x7fffffffLL).to(at::kInt);
}

// A float argument: on main's device, `n` elements, made contiguous fp32.
at::Tensor aux_f32(const at::Tensor& t, const at::Tensor& main, int64_t n, const char* name) {
  require_on(t, main, name);
  TORCH_CHECK(at::isFloatingType(t.scalar_type()), "dsa: ", name, " must be a floating-point tensor");
  require_numel(t, n, name);
  return t.to(at::kFloat).contiguous();
}

c10::optional<at::Tensor> aux_f32(const c10::optional<at::Tensor>& t, const at::Tensor& main, int64_t n,
                                  const char* name) {
  if (!t.has_value()) return t;
  return aux_f32(*t, main, n, name);
}

// A block table [B, max_blocks] (max_blocks >= 1) on main's device, made contiguous int32.
at::Tensor aux_table(const at::Tensor& t, const at::Tensor& main, int64_t B, const char* name) {
  TORCH_CHECK(t.dim() == 2 && t.size(0) == B && t.size(1) > 0, "dsa: ", name, " must be [", B,
              ", max_blocks] (got ", t.sizes(), ")");
  return aux_i32(t, main, -1, name);
}

c10::optional<at::Tensor> aux_table(const c10::optional<at::Tensor>& t, const at::Tensor& main, int64_t B,
                                    const char* name) {
  if (!t.has_value()) return t;
  return aux_table(*t, main, B, name);
}

// ---------------------------------------------------------------- top-k
std::tuple<at::Tensor, at::Tensor> topk_select(const at::Tensor& x, int64_t k, bool sorted) {
  require(x, "x");
  TORCH_CHECK(x.dim() == 2 && x.scalar_type() == at::kFloat, "dsa.topk_select: x must be [rows, n] fp32");
  TORCH_CHECK(k >= 1 && k <= 8192, "dsa.topk_select: k must be in [1, 8192]");
  c10::OptionalDeviceGuard guard(x.device());
  const int64_t rows = x.size(0), n = x.size(1);
  auto idx = at::empty({rows, k}, x.options().dtype(at::kInt));
  auto val = at::empty({rows, k}, x.options());
  const size_t ws_bytes = dsa_topk_select_workspace_size(rows, n, k);
  auto ws = at::empty({(int64_t)(ws_bytes > 0 ? ws_bytes : 1)}, x.options().dtype(at::kByte));
  check_rc(dsa_topk_select_ws(static_cast<const float*>(ptr(x)), n, rows, n, k, nullptr, sorted ? 1 : 0,
                              static_cast<int32_t*>(ptr(idx)), static_cast<float*>(ptr(val)), ptr(ws), ws_bytes,
                              stream_of(x)),
           "topk_select");
  return {idx, val};
}

std::tuple<at::Tensor, at::Tensor> topk_select_meta(const at::Tensor& x, int64_t k, bool) {
  return {at::empty({x.size(0), k}, x.options().dtype(at::kInt)), at::empty({x.size(0), k}, x.options())};
}

// ---------------------------------------------------------------- lightning indexer (BSND query)
// query [B, S1, H, D]; key [B, S2, 1, D] or paged [blocks, block_size, 1, D] with block_table, in
// which case s2 (the longest key length) is required.
std::tuple<at::Tensor, at::Tensor> lightning_indexer(const at::Tensor& query, const at::Tensor& key,
                                                     const at::Tensor& weights,
                                                     const c10::optional<at::Tensor>& key_scale,
                                                     const c10::optional<at::Tensor>& actual_seq_lengths_query,
                                                     const c10::optional<at::Tensor>& actual_seq_lengths_key,
                                                     const c10::optional<at::Tensor>& block_table,
                                                     int64_t sparse_count, int64_t sparse_mode, bool return_value,
                                                     int64_t s2) {
  require(query, "query");
  require(key, "key");
  require_on(key, query, "key");
  TORCH_CHECK(query.dim() == 4 && key.dim() == 4, "dsa.lightning_indexer: query and key must be 4-D");
  TORCH_CHECK(key.scalar_type() == query.scalar_type(), "dsa.lightning_indexer: key dtype must equal query dtype");
  TORCH_CHECK(sparse_count >= 1 && sparse_count <= 8192, "dsa.lightning_indexer: sparse_count must be in [1, 8192]");
  c10::OptionalDeviceGuard guard(query.device());
  const int64_t B = query.size(0), S1 = query.size(1), H = query.size(2), D = query.size(3);
  const bool paged = block_table.has_value();
  TORCH_CHECK(key.size(2) == 1 && key.size(3) == D, "dsa.lightning_indexer: key must be [.., .., 1, ", D, "] (got ",
              key.sizes(), ")");
  TORCH_CHECK(paged || key.size(0) == B, "dsa.lightning_indexer: key batch ", key.size(0), " != query batch ", B);
  TORCH_CHECK(!paged || s2 > 0, "dsa.lightning_indexer: paged keys need s2 (the longest key length)");
  const int64_t S2 = paged ? s2 : key.size(1);
  auto w = aux_f32(weights, query, B * S1 * H, "weights");
  // One scale per key row of `key` (contiguous [B, S2] or paged [blocks, block_size]).
  auto ks = aux_f32(key_scale, query, key.size(0) * key.size(1), "key_scale");
  auto aq = aux_i32(actual_seq_lengths_query, query, B, "actual_seq_lengths_query");
  auto ak = aux_i32(actual_seq_lengths_key, query, B, "actual_seq_lengths_key");
  auto bt = aux_table(block_table, query, B, "block_table");
  TORCH_CHECK(!paged || bt->size(1) * key.size(1) >= S2,
              "dsa.lightning_indexer: block_table covers fewer than s2 keys");
  auto idx = at::empty({B, S1, 1, sparse_count}, query.options().dtype(at::kInt));
  auto val = return_value ? at::empty({B, S1, 1, sparse_count}, query.options().dtype(at::kFloat))
                          : at::empty({0}, query.options().dtype(at::kFloat));
  if (B * S1 == 0) return {idx, val};
  // At least 2048 rows past 32768 keys stream the top-k out of the indexer (same output, no full logits).
  const bool fused = S2 > 32768 && B * S1 >= 2048;
  const size_t ws_bytes = fused ? dsa_lightning_indexer_fused_workspace_size(B, S1, S2, sparse_count)
                                : dsa_lightning_indexer_workspace_size(B, S1, S2, sparse_count);
  auto ws = at::empty({(int64_t)(ws_bytes > 0 ? ws_bytes : 1)}, query.options().dtype(at::kByte));
  check_rc((fused ? dsa_lightning_indexer_fused : dsa_lightning_indexer)(kind_of(query), ptr(query), ptr(key), ptr_or_null<float>(ks),
                                 static_cast<float*>(ptr(w)), B, S1, S2, H, D, ptr_or_null<int32_t>(aq),
                                 ptr_or_null<int32_t>(ak), ptr_or_null<int32_t>(bt), paged ? key.size(1) : 0,
                                 paged ? bt->size(1) : 0, (int)sparse_mode, sparse_count,
                                 static_cast<int32_t*>(ptr(idx)), return_value ? static_cast<float*>(ptr(val)) : nullptr,
                                 ptr(ws), ws_bytes, stream_of(query)),
           "lightning_indexer");
  return {idx, val};
}

std::tuple<at::Tensor, at::Tensor> lightning_indexer_meta(const at::Tensor& query, const at::Tensor&,
                                                          const at::Tensor&, const c10::optional<at::Tensor>&,
                                                          const c10::optional<at::Tensor>&,
                                                          const c10::optional<at::Tensor>&,
                                                          const c10::optional<at::Tensor>&, int64_t sparse_count,
                                                          int64_t, bool return_value, int64_t) {
  const int64_t B = query.size(0), S1 = query.size(1);
  auto idx = at::empty({B, S1, 1, sparse_count}, query.options().dtype(at::kInt));
  auto val = return_value ? at::empty({B, S1, 1, sparse_count}, query.options().dtype(at::kFloat))
                          : at::empty({0}, query.options().dtype(at::kFloat));
  return {idx, val};
}

// ---------------------------------------------------------------- sparse MLA (d_qk 576, d_v 512)
// q [B, S, H, 576]; kv [B, Skv, 1, 576] or paged [blocks, block_size, 1, 576]; indices [B, S, 1, topk].
std::tuple<at::Tensor, at::Tensor> sparse_mla_fwd(const at::Tensor& q, const at::Tensor& kv,
                                                  const at::Tensor& indices, double sm_scale,
                                                  const c10::optional<at::Tensor>& block_table,
                                                  const c10::optional<at::Tensor>& actual_seq_lengths_query,
                                                  const c10::optional<at::Tensor>& actual_seq_lengths_kv,
                                                  bool is_causal) {
  require(q, "q");
  require(kv, "kv");
  require(indices, "indices");
  require_on(kv, q, "kv");
  require_on(indices, q, "indices");
  TORCH_CHECK(q.dim() == 4 && q.size(3) == 576, "dsa.sparse_mla_fwd: q must be [B, S, H, 576] (got ", q.sizes(), ")");
  TORCH_CHECK(kv.dim() == 4 && kv.size(2) == 1 && kv.size(3) == 576,
              "dsa.sparse_mla_fwd: kv must be [B, Skv, 1, 576] or [blocks, block_size, 1, 576] (got ", kv.sizes(), ")");
  TORCH_CHECK(kv.scalar_type() == q.scalar_type(), "dsa.sparse_mla_fwd: kv dtype must equal q dtype");
  TORCH_CHECK(indices.scalar_type() == at::kInt, "dsa.sparse_mla_fwd: indices must be int32");
  c10::OptionalDeviceGuard guard(q.device());
  const int64_t B = q.size(0), S = q.size(1), H = q.size(2);
  TORCH_CHECK(indices.dim() == 4 && indices.size(0) == B && indices.size(1) == S && indices.size(2) == 1 &&
                  indices.size(3) >= 1,
              "dsa.sparse_mla_fwd: indices must be [", B, ", ", S, ", 1, topk] (got ", indices.sizes(), ")");
  const int64_t topk = indices.size(3);
  const bool paged = block_table.has_value();
  TORCH_CHECK(paged || kv.size(0) == B, "dsa.sparse_mla_fwd: kv batch ", kv.size(0), " != q batch ", B);
  auto bt = aux_table(block_table, q, B, "block_table");
  auto aq = aux_i32(actual_seq_lengths_query, q, B, "actual_seq_lengths_query");
  auto ak = aux_i32(actual_seq_lengths_kv, q, B, "actual_seq_lengths_kv");
  auto out = at::empty({B, S, H, 512}, q.options());
  auto lse = at::empty({B, S, H}, q.options().dtype(at::kFloat));
  const size_t ws_bytes = dsa_sparse_mla_workspace_size(B, S, H, topk);
  auto ws = at::empty({(int64_t)(ws_bytes > 0 ? ws_bytes : 1)}, q.options().dtype(at::kByte));
  const int64_t nblk = paged ? bt->size(1) : 0, bs = paged ? kv.size(1) : 0;
  check_rc(dsa_sparse_mla_fwd(kind_of(q), ptr(q), ptr(kv), static_cast<const int32_t*>(ptr(indices)),
                              ptr_or_null<int32_t>(bt), ptr_or_null<int32_t>(aq), ptr_or_null<int32_t>(ak), B, S, H,
                              576, 512, paged ? nblk * bs : kv.size(1), bs, nblk, topk, (float)sm_scale,
                              is_causal ? 1 : 0, ptr(out), static_cast<float*>(ptr(lse)), ptr(ws), ws_bytes,
                              stream_of(q)),
           "sparse_mla_fwd");
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> sparse_mla_fwd_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&,
                                                       double, const c10::optional<at::Tensor>&,
                                                       const c10::optional<at::Tensor>&,
                                                       const c10::optional<at::Tensor>&, bool) {
  return {at::empty({q.size(0), q.size(1), q.size(2), 512}, q.options()),
          at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat))};
}

// ---------------------------------------------------------------- V4 sparse flash MLA (TND rows)
// q [T, H, 512]; q_start / q_len / seqused_kv [B]; caches [blocks, block_size, 1, 512] (or 3-D).
// "hca" (cmp_kv without cmp_sparse_indices) needs max_cmp, the compressed-row bound
// seqused_kv.max() // cmp_ratio that the reference API derives on the host
// (sparse_flash_mla_api.py:177): rows past it would be dropped, so it has no default.
std::tuple<at::Tensor, at::Tensor> sparse_flash_mla(
    const at::Tensor& q, const at::Tensor& ori_kv, const at::Tensor& ori_block_table, const at::Tensor& q_start,
    const at::Tensor& q_len, const at::Tensor& seqused_kv, const c10::optional<at::Tensor>& sinks,
    double softmax_scale, const c10::optional<at::Tensor>& cmp_kv, const c10::optional<at::Tensor>& cmp_block_table,
    const c10::optional<at::Tensor>& cmp_sparse_indices, int64_t cmp_ratio, int64_t ori_win_left, int64_t max_cmp) {
  require(q, "q");
  require(ori_kv, "ori_kv");
  require_on(ori_kv, q, "ori_kv");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == 512, "dsa.sparse_flash_mla: q must be [T, H, 512] (got ", q.sizes(), ")");
  auto check_cache = [&](const at::Tensor& c, const char* name) {
    TORCH_CHECK((c.dim() == 4 && c.size(2) == 1 && c.size(3) == 512) || (c.dim() == 3 && c.size(2) == 512),
                "dsa.sparse_flash_mla: ", name, " must be [blocks, block_size, 1, 512] (got ", c.sizes(), ")");
    TORCH_CHECK(c.scalar_type() == q.scalar_type(), "dsa.sparse_flash_mla: ", name, " dtype must equal q dtype");
  };
  check_cache(ori_kv, "ori_kv");
  c10::OptionalDeviceGuard guard(q.device());
  const int64_t T = q.size(0), H = q.size(1), B = q_start.numel();
  TORCH_CHECK(B >= 1, "dsa.sparse_flash_mla: q_start must have one entry per batch");
  auto obt = aux_table(ori_block_table, q, B, "ori_block_table");
  auto qs = aux_i32(q_start, q, B, "q_start");
  auto ql = aux_i32(q_len, q, B, "q_len");
  auto kl = aux_i32(seqused_kv, q, B, "seqused_kv");
  auto sk = aux_f32(sinks, q, H, "sinks");
  c10::optional<at::Tensor> cbt, idx;
  int64_t K = 0, cmp_slots = 0;
  if (cmp_kv.has_value()) {
    require(*cmp_kv, "cmp_kv");
    require_on(*cmp_kv, q, "cmp_kv");
    check_cache(*cmp_kv, "cmp_kv");
    TORCH_CHECK(cmp_block_table.has_value(), "dsa.sparse_flash_mla: cmp_kv needs cmp_block_table");
    cbt = aux_table(cmp_block_table, q, B, "cmp_block_table");
    if (cmp_sparse_indices.has_value()) {
      const auto& ci = *cmp_sparse_indices;
      TORCH_CHECK(ci.dim() >= 2 && ci.size(0) == T && ci.size(-1) >= 1 && ci.numel() == T * ci.size(-1),
                  "dsa.sparse_flash_mla: cmp_sparse_indices must be [T, (1,) topk_cmp] (got ", ci.sizes(), ")");
      idx = aux_i32(cmp_sparse_indices, q, -1, "cmp_sparse_indices");
      K = ci.size(-1);
      cmp_slots = K;
    } else {
      TORCH_CHECK(max_cmp >= 0, "dsa.sparse_flash_mla: cmp_kv without cmp_sparse_indices needs max_cmp "
                  "(seqused_kv.max() // cmp_ratio)");
      cmp_slots = max_cmp;
    }
  } else {
    TORCH_CHECK(!cmp_sparse_indices.has_value(), "dsa.sparse_flash_mla: cmp_sparse_indices without cmp_kv");
  }
  auto out = at::empty({T, H, 512}, q.options());
  auto lse = at::empty({T, H}, q.options().dtype(at::kFloat));
  const size_t ws_bytes = dsa_sparse_flash_mla_workspace_size(T, H, ori_win_left, cmp_slots);
  auto ws = at::empty({(int64_t)(ws_bytes > 0 ? ws_bytes : 1)}, q.options().dtype(at::kByte));
  const at::Tensor* c = cmp_kv.has_value() ? &*cmp_kv : nullptr;
  check_rc(dsa_sparse_flash_mla(kind_of(q), ptr(q), T, H, 512, B, static_cast<int32_t*>(ptr(qs)),
                                static_cast<int32_t*>(ptr(ql)), static_cast<int32_t*>(ptr(kl)), ptr(ori_kv),
                                ori_kv.size(0), ori_kv.size(1), static_cast<int32_t*>(ptr(obt)), obt.size(1),
                                c ? ptr(*c) : nullptr, c ? c->size(0) : 0, c ? c->size(1) : 0,
                                ptr_or_null<int32_t>(cbt), cbt.has_value() ? cbt->size(1) : 0,
                                ptr_or_null<int32_t>(idx), K, cmp_ratio, ori_win_left, c ? cmp_slots : 0,
                                ptr_or_null<float>(sk), (float)softmax_scale, ptr(out), static_cast<float*>(ptr(lse)),
                                ptr(ws), ws_bytes, stream_of(q)),
           "sparse_flash_mla");
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> sparse_flash_mla_meta(
    const at::Tensor& q, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
    const c10::optional<at::Tensor>&, double, const c10::optional<at::Tensor>&, const c10::optional<at::Tensor>&,
    const c10::optional<at::Tensor>&, int64_t, int64_t, int64_t) {
  return {at::empty({q.size(0), q.size(1), 512}, q.options()),
          at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat))};
}

// ---------------------------------------------------------------- producer
std::tuple<at::Tensor, at::Tensor> act_quant(const at::Tensor& x, bool round_scale,
                                             c10::optional<at::ScalarType> dtype_opt) {
  require(x, "x");
  TORCH_CHECK(x.dim() >= 1, "dsa.act_quant: x must have at least one dimension");
  const at::ScalarType dtype = dtype_opt.value_or(at::kChar);
  TORCH_CHECK(dtype == at::kChar || dtype == at::kFloat8_e4m3fn, "dsa.act_quant: dtype must be int8 or float8_e4m3fn");
  c10::OptionalDeviceGuard guard(x.device());
  const int64_t n = x.size(-1), rows = n ? x.numel() / n : 0;
  auto y = at::empty(x.sizes(), x.options().dtype(dtype));
  auto sizes = x.sizes().vec();
  sizes.back() = 1;
  auto s = at::empty(sizes, x.options().dtype(at::kFloat));
  if (rows * n > 0)
    check_rc(dsa_act_quant(kind_of(x), ptr(x), rows, n, dtype == at::kChar ? DSA_KIND_INT8 : DSA_KIND_FP8_E4M3,
                           ptr(y), static_cast<float*>(ptr(s)), round_scale ? 1 : 0, stream_of(x)),
             "act_quant");
  return {y, s};
}

std::tuple<at::Tensor, at::Tensor> act_quant_meta(const at::Tensor& x, bool, c10::optional<at::ScalarType> dtype_opt) {
  const at::ScalarType dtype = dtype_opt.value_or(at::kChar);
  auto sizes = x.sizes().vec();
  sizes.back() = 1;
  return {at::empty(x.sizes(), x.options().dtype(dtype)), at::empty(sizes, x.options().dtype(at::kFloat))};
}

// V4 gathered-index attention with sinks (examples/deepseek_v4/sparse_attention.py:171-198):
// q [b, m, h, 512], kv [b, n, 512], attn_sink [h] fp32, topk_idxs [b, m, topk] -> (out fp32, lse fp32);
// the kernel writes its fp32 accumulator, as the reference's does.
std::tuple<at::Tensor, at::Tensor> sparse_attn(const at::Tensor& q, const at::Tensor& kv,
                                               const c10::optional<at::Tensor>& attn_sink, const at::Tensor& topk_idxs,
                                               double softmax_scale) {
  require(q, "q");
  require(kv, "kv");
  require_on(kv, q, "kv");
  TORCH_CHECK(q.dim() == 4 && kv.dim() == 3 && topk_idxs.dim() == 3, "dsa.sparse_attn: q [b,m,h,d], kv [b,n,d], "
              "topk_idxs [b,m,topk]");
  TORCH_CHECK(kv.scalar_type() == q.scalar_type(), "dsa.sparse_attn: kv dtype must equal q dtype");
  c10::OptionalDeviceGuard guard(q.device());
  const int64_t B = q.size(0), M = q.size(1), H = q.size(2), D = q.size(3), N = kv.size(1), K = topk_idxs.size(2);
  TORCH_CHECK(kv.size(0) == B && kv.size(2) == D, "dsa.sparse_attn: kv must be [", B, ", n, ", D, "] (got ",
              kv.sizes(), ")");
  TORCH_CHECK(topk_idxs.size(0) == B && topk_idxs.size(1) == M && K >= 1, "dsa.sparse_attn: topk_idxs must be [", B,
              ", ", M, ", topk] (got ", topk_idxs.sizes(), ")");
  auto idx = aux_i32(topk_idxs, q, -1, "topk_idxs");
  auto sk = aux_f32(attn_sink, q, H, "attn_sink");
  auto out = at::empty({B, M, H, D}, q.options().dtype(at::kFloat));
  auto lse = at::empty({B, M, H}, q.options().dtype(at::kFloat));
  if (B * M > 0) {
    const size_t ws_bytes = dsa_sparse_attn_sink_workspace_size(B, M, H, K);
    auto ws = at::empty({(int64_t)(ws_bytes > 0 ? ws_bytes : 1)}, q.options().dtype(at::kByte));
    check_rc(dsa_sparse_attn_sink(kind_of(q), ptr(q), ptr(kv), static_cast<int32_t*>(ptr(idx)), B, M, H, N, D, K,
                                  ptr_or_null<float>(sk), (float)softmax_scale, ptr(out),
                                  static_cast<float*>(ptr(lse)), ptr(ws), ws_bytes, stream_of(q)),
             "sparse_attn");
  }
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> sparse_attn_meta(const at::Tensor& q, const at::Tensor&,
                                                    const c10::optional<at::Tensor>&, const at::Tensor&, double) {
  return {at::empty(q.sizes(), q.options().dtype(at::kFloat)),
          at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat))};
}

// x [..., K] int8, weight [N, K] int8, their row scales, bias [N] -> [..., N] in dtype (bf16 by default).
at::Tensor quant_matmul(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& x_scale,
                        const at::Tensor& weight_scale, const c10::optional<at::Tensor>& bias,
                        c10::optional<at::ScalarType> dtype_opt) {
  require(x, "x");
  require(weight, "weight");
  require_on(weight, x, "weight");
  TORCH_CHECK(x.scalar_type() == at::kChar && weight.scalar_type() == at::kChar,
              "dsa.quant_matmul: x and weight must be int8");
  TORCH_CHECK(x.dim() >= 2 && weight.dim() == 2 && weight.size(1) == x.size(-1),
              "dsa.quant_matmul: x must be [..., K] and weight [N, K] (got ", x.sizes(), ", ", weight.sizes(), ")");
  const at::ScalarType dtype = dtype_opt.value_or(at::kBFloat16);
  TORCH_CHECK(dtype == at::kBFloat16 || dtype == at::kHalf || dtype == at::kFloat,
              "dsa.quant_matmul: dtype must be bfloat16, float16 or float32");
  const int64_t K = x.size(-1), N = weight.size(0);
  TORCH_CHECK(K >= 1 && K <= 131071, "dsa.quant_matmul: K must be in [1, 131071] (got ", K, ")");
  const int64_t M = x.numel() / K;
  c10::OptionalDeviceGuard guard(x.device());
  auto xs = aux_f32(x_scale, x, M, "x_scale");
  auto ws = aux_f32(weight_scale, x, N, "weight_scale");
  auto b = aux_f32(bias, x, N, "bias");
  auto sizes = x.sizes().vec();
  sizes.back() = N;
  auto out = at::empty(sizes, x.options().dtype(dtype));
  if (M > 0 && N > 0) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(ptr(x)) | reinterpret_cast<uintptr_t>(ptr(weight));
    const size_t bytes = dsa_quant_matmul_workspace_size(M, N, K, (at & 15) == 0);
    auto work = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    check_rc(dsa_quant_matmul(kind_of(out), ptr(x), ptr(weight), static_cast<float*>(ptr(xs)),
                              static_cast<float*>(ptr(ws)), ptr_or_null<float>(b), M, N, K, ptr(out),
                              bytes ? ptr(work) : nullptr, bytes, stream_of(x)),
             "quant_matmul");
  }
  return out;
}

at::Tensor quant_matmul_meta(const at::Tensor& x, const at::Tensor& weight, const at::Tensor&, const at::Tensor&,
                             const c10::optional<at::Tensor>&, c10::optional<at::ScalarType> dtype_opt) {
  auto sizes = x.sizes().vec();
  sizes.back() = weight.size(0);
  return at::empty(sizes, x.options().dtype(dtype_opt.value_or(at::kBFloat16)));
}

// Token stride of a [T, n, D] argument whose tokens may lie apart.
int64_t heads_stride(const at::Tensor& t, const at::Tensor& q, const char* name) {
  require_on(t, q, name);
  TORCH_CHECK(t.scalar_type() == q.scalar_type() && t.dim() == 3 && t.size(0) == q.size(0) && t.size(2) == q.size(2) &&
                  t.stride(2) == 1 && (t.size(1) <= 1 || t.stride(1) == t.size(2)),
              "dsa.qk_norm_rope: ", name, " must be [T, heads, D] of one dtype with contiguous heads (got ", t.sizes(),
              ", strides ", t.strides(), ")");
  return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2);
}

void norm_rope(const at::Tensor& q, const at::Tensor& k, const c10::optional<at::Tensor>& v,
               const c10::optional<at::Tensor>& q_weight, const c10::optional<at::Tensor>& k_weight,
               const at::Tensor& positions, const at::Tensor& cos, const at::Tensor& sin,
               const c10::optional<at::Tensor>& slots, double eps, bool interleaved, int64_t rows, at::Tensor& q_out,
               const at::Tensor& k_out, const c10::optional<at::Tensor>& v_out) {
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2), G = k.size(1);
  const int64_t qs = heads_stride(q, q, "q"), ks = heads_stride(k, q, "k"), vs = v ? heads_stride(*v, q, "v") : 0;
  TORCH_CHECK(!v || v->size(1) == G, "dsa.qk_norm_rope: v must have k's heads");
  require_on(cos, q, "cos");
  require_on(sin, q, "sin");
  TORCH_CHECK(cos.dim() == 2 && cos.sizes() == sin.sizes(), "dsa.qk_norm_rope: cos and sin must be [positions, R / 2]");
  auto c = aux_f32(cos, q, cos.numel(), "cos"), s = aux_f32(sin, q, sin.numel(), "sin");
  auto qw = aux_f32(q_weight, q, D, "q_weight"), kw = aux_f32(k_weight, q, D, "k_weight");
  // 64-bit values past 32 bits mark padding.
  auto pos = aux_i32(saturated_i32(positions), q, T, "positions");
  auto at_rows = aux_i32(slots ? c10::make_optional(saturated_i32(*slots)) : slots, q, T, "slots");
  if (T == 0) return;
  check_rc(dsa_qk_norm_rope(kind_of(q), ptr(q), qs, ptr(k), ks, ptr_or_null<void>(v), vs, ptr_or_null<void>(qw),
                            ptr_or_null<void>(kw), DSA_KIND_FP32, static_cast<int32_t*>(ptr(pos)),
                            static_cast<float*>(ptr(c)), static_cast<float*>(ptr(s)), cos.size(0), T, H, G, D,
                            2 * cos.size(1), (float)eps, interleaved ? 1 : 0, ptr_or_null<int32_t>(at_rows), rows,
                            ptr(q_out), ptr(k_out), ptr_or_null<void>(v_out), stream_of(q)),
           "qk_norm_rope");
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope(const at::Tensor& q, const at::Tensor& k,
                                                const c10::optional<at::Tensor>& q_weight,
                                                const c10::optional<at::Tensor>& k_weight, const at::Tensor& positions,
                                                const at::Tensor& cos, const at::Tensor& sin, double eps,
                                                bool interleaved) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && k.dim() == 3, "dsa.qk_norm_rope: q and k must be [T, heads, D] on a device");
  c10::OptionalDeviceGuard guard(q.device());
  auto qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), q.options());
  norm_rope(q, k, c10::nullopt, q_weight, k_weight, positions, cos, sin, c10::nullopt, eps, interleaved, 0, qo, ko,
            c10::nullopt);
  return {qo, ko};
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope_meta(const at::Tensor& q, const at::Tensor& k,
                                                     const c10::optional<at::Tensor>&,
                                                     const c10::optional<at::Tensor>&, const at::Tensor&,
                                                     const at::Tensor&, const at::Tensor&, double, bool) {
  return {at::empty(q.sizes(), q.options()), at::empty(k.sizes(), k.options())};
}

// Keys and values to rows slots[t] of the caches [blocks, block_size, G, D], in place.
at::Tensor qk_norm_rope_paged(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                              const c10::optional<at::Tensor>& q_weight, const c10::optional<at::Tensor>& k_weight,
                              const at::Tensor& positions, const at::Tensor& cos, const at::Tensor& sin,
                              at::Tensor k_cache, at::Tensor v_cache, const at::Tensor& slots, double eps,
                              bool interleaved) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 3 && k.dim() == 3, "dsa.qk_norm_rope: q and k must be [T, heads, D] on a device");
  for (const at::Tensor* c : {&k_cache, &v_cache}) {
    require(*c, "cache");
    require_on(*c, q, "cache");
    TORCH_CHECK(c->dim() == 4 && c->size(2) == k.size(1) && c->size(3) == q.size(2) &&
                    c->scalar_type() == q.scalar_type() && c->sizes() == k_cache.sizes(),
                "dsa.qk_norm_rope_paged: caches must be [blocks, block_size, ", k.size(1), ", ", q.size(2), "] (got ",
                c->sizes(), ")");
  }
  c10::OptionalDeviceGuard guard(q.device());
  auto qo = at::empty(q.sizes(), q.options());
  norm_rope(q, k, v, q_weight, k_weight, positions, cos, sin, slots, eps, interleaved,
            k_cache.size(0) * k_cache.size(1), qo, k_cache, v_cache);
  return qo;
}

at::Tensor qk_norm_rope_paged_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&,
                                   const c10::optional<at::Tensor>&, const c10::optional<at::Tensor>&,
                                   const at::Tensor&, const at::Tensor&, const at::Tensor&, at::Tensor, at::Tensor,
                                   const at::Tensor&, double, bool) {
  return at::empty(q.sizes(), q.options());
}

// q [T, H, D] (actual_seq_lengths_query: inclusive prefix sums) or [B, S, H, D] (lengths, or none).
std::tuple<at::Tensor, at::Tensor> paged_gqa_fwd(const at::Tensor& q, const at::Tensor& k_cache,
                                                 const at::Tensor& v_cache, const at::Tensor& block_table,
                                                 const at::Tensor& actual_seq_lengths_kv, double sm_scale,
                                                 const c10::optional<at::Tensor>& actual_seq_lengths_query,
                                                 bool is_causal, int64_t win_left,
                                                 const c10::optional<at::Tensor>& sinks) {
  require(q, "q");
  require(k_cache, "k_cache");
  require(v_cache, "v_cache");
  require_on(k_cache, q, "k_cache");
  require_on(v_cache, q, "v_cache");
  TORCH_CHECK((q.dim() == 3 || q.dim() == 4) && k_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes() &&
                  k_cache.size(3) == q.size(-1) && block_table.dim() == 2,
              "dsa.paged_gqa_fwd: q [T, H, D] or [B, S, H, D], caches [blocks, block_size, G, D], block_table [B, n]");
  TORCH_CHECK(k_cache.scalar_type() == q.scalar_type() && v_cache.scalar_type() == q.scalar_type(),
              "dsa.paged_gqa_fwd: cache dtypes must equal q dtype");
  const bool packed = q.dim() == 3;
  const int64_t B = block_table.size(0), mb = block_table.size(1), S = packed ? 0 : q.size(1),
                T = packed ? q.size(0) : B * S;
  TORCH_CHECK(packed ? actual_seq_lengths_query.has_value() : q.size(0) == B,
              "dsa.paged_gqa_fwd: packed queries need prefix sums, padded ones one row of block_table per sequence");
  c10::OptionalDeviceGuard guard(q.device());
  // Pages past 32 bits lie outside the pool, lengths past them are cut as smaller ones are.
  auto bt = aux_i32(saturated_i32(block_table), q, -1, "block_table");
  auto kl = aux_i32(saturated_i32(actual_seq_lengths_kv), q, B, "actual_seq_lengths_kv");
  auto ql = aux_i32(actual_seq_lengths_query ? c10::make_optional(saturated_i32(*actual_seq_lengths_query))
                                             : actual_seq_lengths_query,
                    q, B, "actual_seq_lengths_query");
  const int64_t H = q.size(-2), D = q.size(-1), G = k_cache.size(2);
  auto sk = aux_f32(sinks, q, H, "sinks");
  auto out = at::empty(q.sizes(), q.options());
  auto lse = at::empty(q.sizes().slice(0, q.dim() - 1), q.options().dtype(at::kFloat));
  const size_t bytes = dsa_paged_gqa_workspace_size(T, B, H, G, D, mb * k_cache.size(1));
  auto ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
  int32_t* qlp = ptr_or_null<int32_t>(ql);
  check_rc(dsa_paged_gqa_fwd(kind_of(q), ptr(q), ptr(k_cache), ptr(v_cache), static_cast<int32_t*>(ptr(bt)),
                             packed ? qlp : nullptr, packed ? nullptr : qlp, static_cast<int32_t*>(ptr(kl)), T, B, S, H,
                             G, D, k_cache.size(0), k_cache.size(1), mb, is_causal ? 1 : 0, win_left,
                             ptr_or_null<float>(sk), (float)sm_scale, ptr(out), static_cast<float*>(ptr(lse)),
                             bytes ? ptr(ws) : nullptr, bytes, stream_of(q)),
           "paged_gqa_fwd");
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> paged_gqa_fwd_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&,
                                                      const at::Tensor&, const at::Tensor&, double,
                                                      const c10::optional<at::Tensor>&, bool, int64_t,
                                                      const c10::optional<at::Tensor>&) {
  return {at::empty(q.sizes(), q.options()),
          at::empty(q.sizes().slice(0, q.dim() - 1), q.options().dtype(at::kFloat))};
}

}  // namespace

TORCH_LIBRARY(dsa, m) {
  m.def("topk_select(Tensor x, int k, bool sorted=True) -> (Tensor, Tensor)");
  m.def(
      "lightning_indexer(Tensor query, Tensor key, Tensor weights, Tensor? key_scale=None, "
      "Tensor? actual_seq_lengths_query=None, Tensor? actual_seq_lengths_key=None, Tensor? block_table=None, "
      "int sparse_count=2048, int sparse_mode=3, bool return_value=False, int s2=-1) -> (Tensor, Tensor)");
  m.def(
      "sparse_mla_fwd(Tensor q, Tensor kv, Tensor indices, float sm_scale, Tensor? block_table=None, "
      "Tensor? actual_seq_lengths_query=None, Tensor? actual_seq_lengths_kv=None, bool is_causal=True) "
      "-> (Tensor, Tensor)");
  m.def(
      "sparse_flash_mla(Tensor q, Tensor ori_kv, Tensor ori_block_table, Tensor q_start, Tensor q_len, "
      "Tensor seqused_kv, Tensor? sinks, float softmax_scale, Tensor? cmp_kv=None, Tensor? cmp_block_table=None, "
      "Tensor? cmp_sparse_indices=None, int cmp_ratio=4, int ori_win_left=127, int max_cmp=-1) -> (Tensor, Tensor)");
  m.def("act_quant(Tensor x, bool round_scale=False, ScalarType? dtype=None) -> (Tensor, Tensor)");
  m.def(
      "quant_matmul(Tensor x, Tensor weight, Tensor x_scale, Tensor weight_scale, Tensor? bias=None, "
      "ScalarType? dtype=None) -> Tensor");
  m.def(
      "qk_norm_rope(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor positions, Tensor cos, Tensor sin, "
      "float eps=1e-6, bool interleaved=False) -> (Tensor, Tensor)");
  m.def(
      "qk_norm_rope_paged(Tensor q, Tensor k, Tensor v, Tensor? q_weight, Tensor? k_weight, Tensor positions, "
      "Tensor cos, Tensor sin, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slots, float eps=1e-6, "
      "bool interleaved=False) -> Tensor");
  m.def(
      "paged_gqa_fwd(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor actual_seq_lengths_kv, "
      "float sm_scale, Tensor? actual_seq_lengths_query=None, bool is_causal=True, int win_left=-1, "
      "Tensor? sinks=None) -> (Tensor, Tensor)");
  m.def("sparse_attn(Tensor q, Tensor kv, Tensor? attn_sink, Tensor topk_idxs, float softmax_scale) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(dsa, CUDA, m) {
  m.impl("topk_select", &topk_select);
  m.impl("lightning_indexer", &lightning_indexer);
  m.impl("sparse_mla_fwd", &sparse_mla_fwd);
  m.impl("sparse_flash_mla", &sparse_flash_mla);
  m.impl("act_quant", &act_quant);
  m.impl("sparse_attn", &sparse_attn);
  m.impl("quant_matmul", &quant_matmul);
  m.impl("qk_norm_rope", &qk_norm_rope);
  m.impl("qk_norm_rope_paged", &qk_norm_rope_paged);
  m.impl("paged_gqa_fwd", &paged_gqa_fwd);
}

TORCH_LIBRARY_IMPL(dsa, Meta, m) {
  m.impl("topk_select", &topk_select_meta);
  m.impl("lightning_indexer", &lightning_indexer_meta);
  m.impl("sparse_mla_fwd", &sparse_mla_fwd_meta);
  m.impl("sparse_flash_mla", &sparse_flash_mla_meta);
  m.impl("act_quant", &act_quant_meta);
  m.impl("sparse_attn", &sparse_attn_meta);
  m.impl("quant_matmul", &quant_matmul_meta);
  m.impl("qk_norm_rope", &qk_norm_rope_meta);
  m.impl("qk_norm_rope_paged", &qk_norm_rope_paged_meta);
  m.impl("paged_gqa_fwd", &paged_gqa_fwd_meta);
}
