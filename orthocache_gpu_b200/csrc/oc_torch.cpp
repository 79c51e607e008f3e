// Compiled Python binding of the hot decode calls (V2 and V3) and of the
// paged-serving operators.
//
// The ctypes path marshals ~30 arguments per call and reads tensor strides
// and pointers from Python, which costs more host time than a short decode
// takes on the GPU.  This module takes the tensors themselves, allocates the
// output with torch, and calls the library's C ABI
// (include/orthocache_b200.h) directly; it adds no GPU code.  The serving
// operators check their arguments here too: ValueError for shapes and sizes,
// TypeError for dtypes, RuntimeError for devices; a step of a small model is a
// few microseconds on the GPU, so they take their arguments by position and
// unpack them without conversions.
#include <c10/core/AutogradState.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <cmath>
#include <cstdint>
#include <limits>
#include <string>
#include <vector>

#include "../../include/orthocache_b200.h"

// Messages are put together without streams: the C++ compiler that builds
// this module may bring a standard library of its own, whose number formatting
// does not work inside a process that has another one loaded.
#define OC_VALUE(cond, ...) TORCH_CHECK_VALUE(cond, text(__VA_ARGS__))
#define OC_TYPE(cond, ...) TORCH_CHECK_TYPE(cond, text(__VA_ARGS__))
#define OC_RUNTIME(cond, ...) TORCH_CHECK(cond, text(__VA_ARGS__))

namespace {

std::string word_of(const char* s) { return s; }
std::string word_of(int64_t x) { return std::to_string(x); }
std::string word_of(int x) { return std::to_string(x); }
std::string word_of(at::ScalarType t) { return c10::toString(t); }
std::string word_of(const at::Device& d) { return d.str(); }
std::string word_of(at::IntArrayRef sizes) {
  std::string s = "[";
  for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
  return s + "]";
}
template <typename... A>
std::string text(const A&... a) {
  std::string s;
  (s.append(word_of(a)), ...);
  return s;
}

int code_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return OC_F32;
    case at::kHalf: return OC_F16;
    case at::kBFloat16: return OC_BF16;
    case at::kFloat8_e4m3fn: return OC_F8E4M3;
    default: OC_RUNTIME(false, "unsupported dtype ", t.scalar_type());
  }
  return -1;
}

void check(int rc, const char* what) {
  OC_RUNTIME(rc == OC_OK, what, ": ", oc_status_string(rc), " (code ", rc, ")");
}

void* ptr_or_null(const c10::optional<at::Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }

// q (H, hd); keys / values (H, S, hd) with a contiguous last dim; returns out (H, hd) in out_dtype.
at::Tensor v2(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, double zeta_max, int64_t num_splits,
              int64_t num_sms, at::ScalarType out_dtype, const c10::optional<at::Tensor>& mask,
              int64_t retained, int64_t status, int64_t ws, int64_t ws_bytes, int64_t stream) {
  const int64_t H = q.size(0), hd = q.size(1), S = k.size(1);
  at::Tensor out = at::empty({H, hd}, q.options().dtype(out_dtype));
  check(oc_fused_attention_v2(q.data_ptr(), code_of(q), q.stride(0), k.data_ptr(), code_of(k), k.stride(0),
                              k.stride(1), v.data_ptr(), code_of(v), v.stride(0), v.stride(1), (int)H, S, (int)hd,
                              zeta_max, (int)num_splits, (int)num_sms, out.data_ptr(), code_of(out), out.stride(0),
                              static_cast<uint8_t*>(ptr_or_null(mask)), reinterpret_cast<uint32_t*>(retained),
                              reinterpret_cast<uint32_t*>(status), reinterpret_cast<void*>(ws), (size_t)ws_bytes,
                              reinterpret_cast<void*>(stream)),
        "fused_orthocache_attention_v2");
  return out;
}

// q (B, Hq, hd); keys / values (B, KVH, S, hd); returns out (B, Hq, hd) in out_dtype.
at::Tensor v3(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, double tau, int64_t group,
              int64_t num_splits, int64_t num_sms, at::ScalarType out_dtype, const c10::optional<at::Tensor>& mask,
              int64_t retained, int64_t status, int64_t ws, int64_t ws_bytes, int64_t stream) {
  const int64_t B = k.size(0), KVH = k.size(1), S = k.size(2), hd = k.size(3);
  at::Tensor out = at::empty({B, KVH * group, hd}, q.options().dtype(out_dtype));
  check(oc_fused_attention_v3_gqa(q.data_ptr(), code_of(q), q.stride(0), q.stride(1), k.data_ptr(), code_of(k),
                                  k.stride(0), k.stride(1), k.stride(2), v.data_ptr(), code_of(v), v.stride(0),
                                  v.stride(1), v.stride(2), (int)B, (int)KVH, (int)group, S, (int)hd, tau,
                                  (int)num_splits, (int)num_sms, out.data_ptr(), code_of(out), out.stride(0),
                                  out.stride(1), static_cast<uint8_t*>(ptr_or_null(mask)),
                                  reinterpret_cast<uint32_t*>(retained), reinterpret_cast<uint32_t*>(status),
                                  reinterpret_cast<void*>(ws), (size_t)ws_bytes, reinterpret_cast<void*>(stream)),
        "fused_orthocache_attention_v3_gqa");
  return out;
}

// ---------------------------------------------------------------- serving operators
using at::Tensor;
using OptTensor = c10::optional<Tensor>;

void need_cuda(const Tensor& t, const Tensor& like) {
  OC_RUNTIME(t.is_cuda(), "orthocache_gpu_b200 runs on CUDA tensors only (no CPU fallback); got a tensor on ",
              t.device());
  OC_RUNTIME(t.device() == like.device(), "tensors on different devices: ", like.device(), " and ", t.device());
}

// Whether forward-mode derivatives are being computed.
bool forward_mode() {
  return c10::AutogradState::get_tls_state().get_fw_grad_mode() && torch::autograd::ForwardADLevel::try_get_by_idx(0);
}

// No derivative is lost without a word: neither a backward pass nor a forward-mode one through this tensor.
void need_constant(const Tensor& t, const char* name, bool forward) {
  if (!t.unsafeGetTensorImpl()->autograd_meta()) return;  // has neither
  OC_RUNTIME(!(t.requires_grad() && at::GradMode::is_enabled()), name,
              " requires grad, and this operator has no backward pass; call it under torch.no_grad()");
  OC_RUNTIME(!(forward && t._fw_grad(0).defined()), name,
              " has a forward-mode derivative, and this operator does not pass it on");
}

// Marks a tensor that a call writes to, as in-place operations of torch do: a backward pass that saved it fails then.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();  // inference tensors have no version
}

// An input of an operator that has no backward pass.
void need_input(const Tensor& t, const Tensor& like, const char* name) {
  need_cuda(t, like);
  need_constant(t, name, forward_mode());
}

int float_code(const Tensor& t, const char* name) {
  const auto s = t.scalar_type();
  OC_TYPE(s == at::kFloat || s == at::kHalf || s == at::kBFloat16, name,
                   " must be float32, float16 or bfloat16, got ", s);
  return code_of(t);
}

// The dtype code of a cache pair: that of the inputs, or float8_e4m3fn for both.
int cache_code(const Tensor& k, const Tensor& v, const Tensor& in) {
  OC_TYPE(k.scalar_type() == v.scalar_type(), "k_cache and v_cache must share a dtype, got ",
                   k.scalar_type(), " and ", v.scalar_type());
  OC_TYPE(k.scalar_type() == in.scalar_type() || k.scalar_type() == at::kFloat8_e4m3fn,
                   "the caches must be of the inputs' dtype (", in.scalar_type(), ") or float8_e4m3fn, got ",
                   k.scalar_type());
  return code_of(k);
}

Tensor rows(const Tensor& t) { return t.dim() == 0 || t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.contiguous(); }

Tensor ints(const Tensor& t, const Tensor& like, const char* name) {
  need_cuda(t, like);
  OC_TYPE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64, got ",
                   t.scalar_type());
  return rows(t.scalar_type() == at::kInt ? t : t.to(at::kInt));
}

Tensor floats(const Tensor& t, const Tensor& like, const char* name) {
  need_input(t, like, name);
  OC_TYPE(t.scalar_type() == at::kFloat, name, " must be float32, got ", t.scalar_type());
  return t.contiguous();
}

int as_int(int64_t x, const char* name) {
  OC_VALUE(x >= 0 && x <= std::numeric_limits<int>::max(), name, " (", x, ") is out of range");
  return static_cast<int>(x);
}

// k_cache / v_cache (num_blocks, kv_heads, block_size, head_dim)
void need_cache(const Tensor& k, const Tensor& v, const Tensor& like, int64_t kv_heads, int64_t head_dim) {
  need_input(k, like, "k_cache");
  need_input(v, like, "v_cache");
  OC_VALUE(k.dim() == 4 && k.sizes() == v.sizes(),
                    "k_cache and v_cache must be (num_blocks, kv_heads, block_size, head_dim) alike, got ", k.sizes(),
                    " and ", v.sizes());
  OC_VALUE(k.size(3) == head_dim, "the caches' head_dim (", k.size(3), ") is not the inputs' (", head_dim, ")");
  OC_VALUE(kv_heads < 0 || k.size(1) == kv_heads, "the caches' kv_heads (", k.size(1),
                    ") is not that of k (", kv_heads, ")");
  OC_VALUE(k.stride(3) == 1 && v.stride(3) == 1, "the caches' last dimension must be contiguous");
  const int64_t bs = k.size(2);
  OC_VALUE(bs > 0 && (bs & (bs - 1)) == 0, "block_size (", bs, ") must be a power of 2");
}

Tensor need_tables(const Tensor& t, const Tensor& like) {
  OC_VALUE(t.dim() == 2, "block_tables must be (num_seqs, max_blocks), got ", t.sizes());
  return ints(t, like, "block_tables");
}

uint32_t* word(int64_t p) { return reinterpret_cast<uint32_t*>(p); }
void* handle(int64_t p) { return reinterpret_cast<void*>(p); }

// q (T, Hq, D); returns (q_out or None, k_out or None)
std::tuple<OptTensor, OptTensor> rotary_append(const OptTensor& q_, const OptTensor& k_, const OptTensor& v_,
                                               const Tensor& positions_, const OptTensor& cos_, const OptTensor& sin_,
                                               const OptTensor& k_cache, const OptTensor& v_cache,
                                               const OptTensor& tables_, const OptTensor& seq_ids_, bool interleaved,
                                               bool inverse, double k_scale, double v_scale, bool return_keys,
                                               int64_t num_sms, int64_t status, int64_t stream) {
  OC_VALUE(q_.has_value() || k_.has_value(), "give q, k or both");
  const Tensor& like = q_.has_value() ? *q_ : *k_;
  need_cuda(like, like);
  const c10::DeviceGuard guard(like.device());
  oc_rotary_args a = {};
  a.dtype = float_code(like, "q");
  OC_VALUE(like.dim() == 3, "q and k must be (tokens, heads, head_dim), got ", like.sizes());
  const int64_t T = like.size(0), D = like.size(2);
  a.tokens = T;
  a.head_dim = as_int(D, "head_dim");
  Tensor q, k, v, pos, cos, sin, tables, seq_ids;
  OptTensor q_out, k_out;
  auto part = [&](const Tensor& t, const char* name) {
    need_input(t, like, name);
    OC_TYPE(t.scalar_type() == like.scalar_type(), name, " must be ", like.scalar_type(), ", got ",
                     t.scalar_type());
    OC_VALUE(t.dim() == 3 && t.size(0) == T && t.size(2) == D, name, " must be (", T, ", heads, ", D,
                      "), got ", t.sizes());
    return rows(t);
  };
  if (q_.has_value()) {
    q = part(*q_, "q");
    q_out = at::empty(q.sizes(), q.options());
    a.q = q.data_ptr();
    a.q_tok_stride = q.stride(0);
    a.q_head_stride = q.stride(1);
    a.q_heads = as_int(q.size(1), "q_heads");
    a.q_out = q_out->data_ptr();
    a.qo_tok_stride = q_out->stride(0);
    a.qo_head_stride = q_out->stride(1);
  }
  OC_VALUE(positions_.dim() == 1 && positions_.size(0) == T, "positions must be (", T, ",), got ",
                    positions_.sizes());
  need_cuda(positions_, like);
  OC_TYPE(positions_.scalar_type() == at::kInt || positions_.scalar_type() == at::kLong,
                   "positions must be int32 or int64, got ", positions_.scalar_type());
  pos = positions_.contiguous();
  a.positions = pos.data_ptr();
  a.positions_64 = pos.scalar_type() == at::kLong;
  OC_VALUE(cos_.has_value() == sin_.has_value(), "give cos and sin together");
  if (cos_.has_value()) {
    cos = floats(*cos_, like, "cos");
    sin = floats(*sin_, like, "sin");
    OC_VALUE(cos.dim() == 2 && cos.sizes() == sin.sizes() && 2 * cos.size(1) <= D,
                      "cos and sin must be (positions, rotary_dim / 2) with rotary_dim <= head_dim (", D, "), got ",
                      cos.sizes(), " and ", sin.sizes());
    a.cos_tab = cos.data_ptr<float>();
    a.sin_tab = sin.data_ptr<float>();
    a.table_rows = cos.size(0);
    a.rotary_dim = 2 * (int)cos.size(1);
    OC_VALUE(T == 0 || a.table_rows > 0, "cos and sin have no rows");
  }
  if (k_.has_value()) {
    k = part(*k_, "k");
    a.k = k.data_ptr();
    a.k_tok_stride = k.stride(0);
    a.k_head_stride = k.stride(1);
    a.kv_heads = as_int(k.size(1), "kv_heads");
    if (return_keys || !k_cache.has_value()) {
      k_out = at::empty(k.sizes(), k.options());
      a.k_out = k_out->data_ptr();
      a.ko_tok_stride = k_out->stride(0);
      a.ko_head_stride = k_out->stride(1);
    }
  }
  OC_VALUE(k_cache.has_value() == v_cache.has_value() && k_cache.has_value() == tables_.has_value() &&
                        k_cache.has_value() == v_.has_value(),
                    "give v, k_cache, v_cache and block_tables together");
  if (k_cache.has_value()) {
    OC_VALUE(k_.has_value(), "give k with the caches");
    v = part(*v_, "v");
    OC_VALUE(v.size(1) == k.size(1), "v must have k's heads (", k.size(1), "), got ", v.size(1));
    need_cache(*k_cache, *v_cache, like, k.size(1), D);
    a.cache_dtype = cache_code(*k_cache, *v_cache, like);
    OC_VALUE(a.cache_dtype == OC_F8E4M3 || (k_scale == 1.0 && v_scale == 1.0),
                      "k_scale and v_scale belong to float8 caches");
    OC_VALUE(k_scale > 0 && v_scale > 0, "k_scale and v_scale must be positive");
    tables = need_tables(*tables_, like);
    a.v = v.data_ptr();
    a.v_tok_stride = v.stride(0);
    a.v_head_stride = v.stride(1);
    a.k_cache = k_cache->data_ptr();
    a.v_cache = v_cache->data_ptr();
    a.num_blocks = k_cache->size(0);
    a.block_size = as_int(k_cache->size(2), "block_size");
    a.kc_block_stride = k_cache->stride(0);
    a.kc_head_stride = k_cache->stride(1);
    a.kc_tok_stride = k_cache->stride(2);
    a.vc_block_stride = v_cache->stride(0);
    a.vc_head_stride = v_cache->stride(1);
    a.vc_tok_stride = v_cache->stride(2);
    a.block_tables = tables.data_ptr<int32_t>();
    a.block_table_stride = tables.stride(0);
    a.num_seqs = as_int(tables.size(0), "num_seqs");
    a.max_blocks = as_int(tables.size(1), "max_blocks");
    a.k_scale = (float)k_scale;
    a.v_scale = (float)v_scale;
    if (seq_ids_.has_value()) {
      OC_VALUE(seq_ids_->dim() == 1 && seq_ids_->size(0) == T, "seq_ids must be (", T, ",), got ",
                        seq_ids_->sizes());
      seq_ids = ints(*seq_ids_, like, "seq_ids");
      a.seq_ids = seq_ids.data_ptr<int32_t>();
    } else {
      OC_VALUE(T == a.num_seqs, "without seq_ids there must be one token per sequence: ", T, " tokens, ",
                        a.num_seqs, " sequences");
    }
    // an empty table or cache has no storage to point to, and no slot either
    if (a.k_cache == nullptr || a.block_tables == nullptr) {
      OC_VALUE(T == 0, "the caches or block_tables are empty");
    }
  }
  a.flags = (interleaved ? OC_ROTARY_INTERLEAVED : 0) | (inverse ? OC_ROTARY_INVERSE : 0);
  a.num_sms = (int)num_sms;
  a.status = word(status);
  if (T > 0 && D > 0) check(oc_rotary_append_paged(&a, handle(stream)), "rotary_append_paged");
  if (k_cache.has_value()) {
    written(*k_cache);
    written(*v_cache);
  }
  return {q_out, k_out};
}

// q (S, Hq, D); returns (out, lse or None)
std::tuple<Tensor, OptTensor> paged_decode(const Tensor& q_, const Tensor& k_cache, const Tensor& v_cache,
                                           const Tensor& tables_, const Tensor& seq_lens_, double scale,
                                           double softcap, const OptTensor& slopes_, int64_t window, double k_scale,
                                           double v_scale, bool return_lse, int64_t num_sms, int64_t status,
                                           int64_t stream) {
  need_input(q_, q_, "q");
  const c10::DeviceGuard guard(q_.device());
  oc_paged_decode_args a = {};
  a.dtype = float_code(q_, "q");
  OC_VALUE(q_.dim() == 3, "q must be (num_seqs, heads, head_dim), got ", q_.sizes());
  const int64_t S = q_.size(0), H = q_.size(1), D = q_.size(2);
  need_cache(k_cache, v_cache, q_, -1, D);
  a.cache_dtype = cache_code(k_cache, v_cache, q_);
  OC_VALUE(a.cache_dtype == OC_F8E4M3 || (k_scale == 1.0 && v_scale == 1.0),
                    "k_scale and v_scale belong to float8 caches");
  const int64_t HK = k_cache.size(1);
  OC_VALUE(HK > 0 && H % HK == 0 && H > 0, "the query heads (", H, ") must be a multiple of the kv heads (",
                    HK, ")");
  OC_VALUE(D > 0 && D <= 256, "head_dim (", D, ") must be between 1 and 256");
  OC_VALUE(softcap >= 0, "softcap must not be negative");
  const Tensor q = rows(q_), tables = need_tables(tables_, q);
  OC_VALUE(tables.size(0) == S, "block_tables must have one row per sequence (", S, "), got ",
                    tables.size(0));
  OC_VALUE(seq_lens_.dim() == 1 && seq_lens_.size(0) == S, "seq_lens must be (", S, ",), got ",
                    seq_lens_.sizes());
  const Tensor lens = ints(seq_lens_, q, "seq_lens");
  Tensor slopes;
  if (slopes_.has_value()) {
    slopes = floats(*slopes_, q, "alibi_slopes");
    OC_VALUE(slopes.dim() == 1 && slopes.size(0) == H, "alibi_slopes must be (", H, ",), got ",
                      slopes.sizes());
    a.slopes = slopes.data_ptr<float>();
  }
  Tensor out = at::empty({S, H, D}, q.options());
  OptTensor lse;
  if (return_lse) {
    lse = at::empty({S, H}, q.options().dtype(at::kFloat));
    a.lse = lse->data_ptr<float>();
  }
  if (S == 0) return {out, lse};
  a.q = q.data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.out = out.data_ptr();
  a.block_tables = tables.data_ptr<int32_t>();
  a.seq_lens = lens.data_ptr<int32_t>();
  a.q_seq_stride = q.stride(0);
  a.q_head_stride = q.stride(1);
  a.out_seq_stride = out.stride(0);
  a.out_head_stride = out.stride(1);
  a.kc_block_stride = k_cache.stride(0);
  a.kc_head_stride = k_cache.stride(1);
  a.kc_tok_stride = k_cache.stride(2);
  a.vc_block_stride = v_cache.stride(0);
  a.vc_head_stride = v_cache.stride(1);
  a.vc_tok_stride = v_cache.stride(2);
  a.block_table_stride = tables.stride(0);
  a.num_blocks = k_cache.size(0);
  a.status = word(status);
  a.scale = (float)scale;
  a.softcap = (float)softcap;
  a.k_scale = (float)k_scale;
  a.v_scale = (float)v_scale;
  a.num_seqs = as_int(S, "num_seqs");
  a.kv_heads = as_int(HK, "kv_heads");
  a.group = (int)(H / HK);
  a.head_dim = (int)D;
  a.block_size = as_int(k_cache.size(2), "block_size");
  a.max_blocks = a.num_blocks ? as_int(tables.size(1), "max_blocks") : 0;
  a.window = as_int(window, "window");
  a.num_sms = (int)num_sms;
  // per call from torch's allocator: calls on other streams, and captured graphs, have their own
  Tensor space;
  a.workspace_bytes = oc_paged_decode_workspace_bytes(&a);
  if (a.workspace_bytes) {
    space = at::empty({(int64_t)a.workspace_bytes}, q.options().dtype(at::kByte));
    a.workspace = space.data_ptr();
  }
  check(oc_paged_decode_attention(&a, handle(stream)), "paged_decode_attention");
  return {out, lse};
}

// q (T, Hq, D), k / v (Tk, Hk, D); returns (out, lse or None)
std::tuple<Tensor, OptTensor> prompt(const Tensor& q_, const Tensor& k_, const Tensor& v_, const OptTensor& cu_q_,
                                     const OptTensor& cu_k_, bool causal, const OptTensor& prefix_, int64_t window,
                                     double scale, double softcap, const OptTensor& slopes_, bool return_lse,
                                     int64_t num_sms, int64_t status, int64_t stream) {
  need_input(q_, q_, "q");
  need_input(k_, q_, "k");
  need_input(v_, q_, "v");
  const c10::DeviceGuard guard(q_.device());
  oc_prompt_args a = {};
  a.dtype = float_code(q_, "q");
  OC_TYPE(k_.scalar_type() == q_.scalar_type() && v_.scalar_type() == q_.scalar_type(),
                   "k and v must be of q's dtype (", q_.scalar_type(), "), got ", k_.scalar_type(), " and ",
                   v_.scalar_type());
  OC_VALUE(q_.dim() == 3 && k_.dim() == 3 && k_.sizes() == v_.sizes() && k_.size(2) == q_.size(2),
                    "q must be (tokens, heads, head_dim), k and v (key tokens, kv heads, head_dim) alike, got ",
                    q_.sizes(), ", ", k_.sizes(), " and ", v_.sizes());
  const int64_t T = q_.size(0), H = q_.size(1), D = q_.size(2), TK = k_.size(0), HK = k_.size(1);
  OC_VALUE(HK > 0 && H > 0 && H % HK == 0, "the query heads (", H, ") must be a multiple of the kv heads (",
                    HK, ")");
  OC_VALUE(D > 0 && D <= (q_.scalar_type() == at::kFloat ? 256 : 128) &&
                        (D % 8 == 0 || q_.scalar_type() == at::kFloat),
                    "head_dim (", D, ") must be a multiple of 8 up to 128, or up to 256 in float32");
  OC_VALUE(softcap >= 0, "softcap must not be negative");
  const Tensor q = rows(q_), k = rows(k_), v = rows(v_);
  OC_VALUE(cu_q_.has_value() || !cu_k_.has_value(), "give cu_seqlens with cu_seqlens_k");
  Tensor cu_q, cu_k, prefix, slopes;
  if (cu_q_.has_value()) {
    cu_q = ints(*cu_q_, q, "cu_seqlens");
    OC_VALUE(cu_q.dim() == 1 && cu_q.size(0) >= 1, "cu_seqlens must be (documents + 1,), got ", cu_q.sizes());
    OC_VALUE(cu_k_.has_value() || TK == T, "without cu_seqlens_k there must be as many keys (", TK,
                      ") as queries (", T, ")");
    a.docs = as_int(cu_q.size(0) - 1, "documents");
    a.cu_q = cu_q.data_ptr<int32_t>();
    a.cu_k = a.cu_q;
    if (cu_k_.has_value()) {
      cu_k = ints(*cu_k_, q, "cu_seqlens_k");
      OC_VALUE(cu_k.dim() == 1 && cu_k.size(0) == cu_q.size(0), "cu_seqlens_k must be (", cu_q.size(0),
                        ",), got ", cu_k.sizes());
      a.cu_k = cu_k.data_ptr<int32_t>();
    }
  } else {
    a.docs = 1;  // one document: all queries over all keys
  }
  if (prefix_.has_value()) {
    prefix = ints(*prefix_, q, "prefix_lens");
    OC_VALUE(prefix.dim() == 1 && prefix.size(0) == a.docs, "prefix_lens must be (", a.docs, ",), got ",
                      prefix.sizes());
    a.prefix_lens = prefix.data_ptr<int32_t>();
  }
  if (slopes_.has_value()) {
    slopes = floats(*slopes_, q, "alibi_slopes");
    OC_VALUE(slopes.dim() == 1 && slopes.size(0) == H, "alibi_slopes must be (", H, ",), got ",
                      slopes.sizes());
    a.slopes = slopes.data_ptr<float>();
  }
  Tensor out = at::empty({T, H, D}, q.options());
  OptTensor lse;
  if (return_lse) {
    lse = at::empty({T, H}, q.options().dtype(at::kFloat));
    a.lse = lse->data_ptr<float>();
    a.lse_tok_stride = H;
  }
  if (T == 0) return {out, lse};
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.out = out.data_ptr();
  a.q_tok_stride = q.stride(0);
  a.q_head_stride = q.stride(1);
  a.k_tok_stride = k.stride(0);
  a.k_head_stride = k.stride(1);
  a.v_tok_stride = v.stride(0);
  a.v_head_stride = v.stride(1);
  a.out_tok_stride = out.stride(0);
  a.out_head_stride = out.stride(1);
  a.tokens = T;
  a.key_tokens = TK;
  a.status = word(status);
  a.scale = (float)scale;
  a.softcap = (float)softcap;
  a.kv_heads = as_int(HK, "kv_heads");
  a.group = (int)(H / HK);
  a.head_dim = (int)D;
  a.causal = causal;
  a.window = as_int(window, "window");
  a.num_sms = (int)num_sms;
  check(oc_prompt_attention(&a, handle(stream)), "prompt_attention");
  return {out, lse};
}

// ---------------------------------------------------------------- pages
struct CacheList {
  std::vector<void*> base;
  std::vector<int64_t> stride;
  std::vector<at::TensorImpl*> all;  // the tensors of the caller's list, which outlive the call
  int64_t page_bytes = 1, num_pages = 0;

  // a list or tuple of tensors, looked at without a conversion: a model has tens of caches, a call a few us
  CacheList(py::handle caches, const Tensor& like) {
    const bool list = PyList_Check(caches.ptr());
    OC_TYPE(list || PyTuple_Check(caches.ptr()), "caches must be a list or tuple of tensors");
    const Py_ssize_t n = list ? PyList_GET_SIZE(caches.ptr()) : PyTuple_GET_SIZE(caches.ptr());
    base.reserve(n);
    stride.reserve(n);
    all.reserve(n);
    const Tensor* first = nullptr;
    const bool forward = forward_mode();
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = list ? PyList_GET_ITEM(caches.ptr(), i) : PyTuple_GET_ITEM(caches.ptr(), i);
      OC_TYPE(THPVariable_Check(o), "caches must be a list or tuple of tensors");
      const Tensor& c = THPVariable_Unpack(o);
      need_cuda(c, like);
      need_constant(c, "a cache", forward);
      if (!first || c.scalar_type() != first->scalar_type() || c.sizes() != first->sizes() ||
          c.strides() != first->strides()) {
        OC_VALUE(c.dim() >= 2, "a cache must be (num_blocks, ...), got ", c.sizes());
        const int64_t es = c.element_size(), pages = c.size(0);
        const int64_t bytes = pages ? c.numel() / pages * es : 0;
        bool dense = bytes > 0 && c.stride(0) * es >= bytes;  // a page of contiguous elements
        for (int64_t d = c.dim() - 1, run = 1; dense && d > 0; run *= c.size(d--))
          dense = c.size(d) == 1 || c.stride(d) == run;
        OC_VALUE(pages == 0 || dense, "a page of a cache must be contiguous, got strides ", c.strides());
        OC_VALUE(!first || (pages == num_pages && (pages == 0 || bytes == page_bytes)),
                          "the caches must have pages of one size and number");
        num_pages = pages;
        if (pages) page_bytes = bytes;
        first = &c;
      }
      all.push_back(c.unsafeGetTensorImpl());
      base.push_back(c.data_ptr());
      stride.push_back(c.stride(0) * (int64_t)c.element_size());
    }
    if (num_pages == 0) base.clear();  // nothing to move
  }
  int count() const { return static_cast<int>(base.size()); }
  void written() const {
    for (at::TensorImpl* t : all)
      if (!t->is_inference()) t->bump_version();
  }
};

Tensor need_int32(const Tensor& t, const Tensor& like, const char* name, int64_t dim) {
  need_cuda(t, like);
  OC_TYPE(t.scalar_type() == at::kInt, name, " must be int32, got ", t.scalar_type());
  OC_VALUE(t.dim() == dim && (t.numel() == 0 || t.stride(-1) == 1), name, " must have ", dim,
                    " dimensions, the last contiguous");
  return t;
}

void need_len(const Tensor& t, int64_t n, const char* name) {
  OC_VALUE(t.size(0) == n, name, " must be (", n, ",), got ", t.sizes());
}

void copy_pages(py::handle caches, const Tensor& src_, const Tensor& dst_, int64_t num_sms,
                int64_t status, int64_t stream) {
  need_cuda(src_, src_);
  const c10::DeviceGuard guard(src_.device());
  const Tensor src = ints(src_, src_, "src"), dst = ints(dst_, src_, "dst");
  OC_VALUE(src.dim() == 1 && src.sizes() == dst.sizes(), "src and dst must be (pairs,) alike, got ",
                    src.sizes(), " and ", dst.sizes());
  const CacheList c(caches, src);
  if (src.numel() == 0 || c.count() == 0) return;
  check(oc_copy_pages(c.base.data(), c.stride.data(), c.count(), c.page_bytes, c.num_pages, src.data_ptr<int32_t>(),
                      dst.data_ptr<int32_t>(), src.numel(), word(status), (int)num_sms, handle(stream)),
        "copy_pages");
  c.written();
}

std::tuple<Tensor, Tensor, Tensor> fork_sequences(const Tensor& tables, const Tensor& lens, const Tensor& refs,
                                                  const Tensor& source_, int64_t block_size, int64_t status,
                                                  int64_t stream) {
  need_int32(tables, tables, "block_tables", 2);
  const c10::DeviceGuard guard(tables.device());
  need_int32(lens, tables, "seq_lens", 1);
  need_int32(refs, tables, "refcounts", 1);
  const int64_t S = tables.size(0);
  need_len(lens, S, "seq_lens");
  OC_VALUE(source_.dim() == 1, "source must be (", S, ",), got ", source_.sizes());
  need_len(source_, S, "source");
  const Tensor source = ints(source_, tables, "source");
  OC_VALUE(block_size > 0, "block_size (", block_size, ") must be positive");
  Tensor t = at::empty({S, tables.size(1)}, tables.options()), l = at::empty({S}, lens.options()),
         r = at::empty({refs.size(0)}, refs.options());
  check(oc_fork_sequences(tables.data_ptr<int32_t>(), tables.stride(0), t.data_ptr<int32_t>(), t.stride(0),
                          lens.data_ptr<int32_t>(), l.data_ptr<int32_t>(), refs.data_ptr<int32_t>(),
                          r.data_ptr<int32_t>(), source.data_ptr<int32_t>(), as_int(S, "num_seqs"),
                          as_int(tables.size(1), "max_blocks"), refs.size(0), as_int(block_size, "block_size"),
                          word(status), handle(stream)),
        "fork_sequences");
  return {t, l, r};
}

// Returns a tensor of one int32 on the device, 1 if the pages were reserved, else 0, where it is asked for.
OptTensor reserve_pages(py::handle caches, const Tensor& tables, const Tensor& lens, const Tensor& refs,
                        const Tensor& wanted_, int64_t block_size, bool return_done, int64_t num_sms, int64_t status,
                        int64_t stream) {
  need_int32(tables, tables, "block_tables", 2);
  const c10::DeviceGuard guard(tables.device());
  need_int32(lens, tables, "seq_lens", 1);
  need_int32(refs, tables, "refcounts", 1);
  const int64_t S = tables.size(0);
  need_len(lens, S, "seq_lens");
  OC_VALUE(wanted_.dim() == 1, "wanted must be (", S, ",), got ", wanted_.sizes());
  need_len(wanted_, S, "wanted");
  const Tensor wanted = ints(wanted_, tables, "wanted");
  OC_VALUE(block_size > 0, "block_size (", block_size, ") must be positive");
  const CacheList c(caches, tables);
  OC_VALUE(c.count() == 0 || c.num_pages == refs.size(0), "the caches have ", c.num_pages,
                    " pages, refcounts ", refs.size(0));
  if (S == 0) return return_done ? OptTensor(at::ones({}, tables.options())) : c10::nullopt;
  const size_t bytes = oc_reserve_workspace_bytes(as_int(S, "num_seqs"), refs.size(0));
  const Tensor space = at::empty({(int64_t)bytes / 4}, tables.options());
  check(oc_reserve_pages(c.base.data(), c.stride.data(), c.count(), c.page_bytes, tables.data_ptr<int32_t>(),
                         tables.stride(0), lens.data_ptr<int32_t>(), refs.data_ptr<int32_t>(),
                         wanted.data_ptr<int32_t>(), (int)S, as_int(tables.size(1), "max_blocks"), refs.size(0),
                         as_int(block_size, "block_size"), space.data_ptr(), bytes, word(status), (int)num_sms,
                         handle(stream)),
        "reserve_pages");
  c.written();
  written(tables);
  written(refs);
  return return_done ? OptTensor(space.select(0, 1)) : c10::nullopt;
}

std::tuple<Tensor, Tensor> compact_pages(py::handle caches, const Tensor& tables, const Tensor& refs,
                                         int64_t num_sms, int64_t status, int64_t stream) {
  need_int32(tables, tables, "block_tables", 2);
  const c10::DeviceGuard guard(tables.device());
  need_int32(refs, tables, "refcounts", 1);
  const CacheList c(caches, tables);
  const int64_t P = refs.size(0);
  OC_VALUE(c.count() == 0 || c.num_pages == P, "the caches have ", c.num_pages, " pages, refcounts ", P);
  Tensor t = at::empty({tables.size(0), tables.size(1)}, tables.options()), r = at::empty({P}, refs.options());
  if (P == 0) return {t.fill_(-1), r};
  const size_t bytes = oc_compact_workspace_bytes(P);
  Tensor space = at::empty({(int64_t)bytes}, tables.options().dtype(at::kByte));
  check(oc_compact_pages(c.base.data(), c.stride.data(), c.count(), c.page_bytes, tables.data_ptr<int32_t>(),
                         tables.stride(0), t.data_ptr<int32_t>(), t.stride(0), refs.data_ptr<int32_t>(),
                         r.data_ptr<int32_t>(), as_int(tables.size(0), "num_seqs"),
                         as_int(tables.size(1), "max_blocks"), P, space.data_ptr(), bytes, word(status), (int)num_sms,
                         handle(stream)),
        "compact_pages");
  c.written();
  return {t, r};
}

// ---------------------------------------------------------------- entry points of the serving operators
struct Context {
  int64_t num_sms = 0, status = 0, stream = 0;
};

// The library's status word on a device.  One word for all streams: a captured call reports to the same place as an
// eager one, whichever stream replays it, and nothing that a stream owns has to outlive it.
uint32_t* status_of(int64_t device) {
  const c10::DeviceGuard guard(c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(device)));
  uint32_t* w = nullptr;
  check(oc_device_status(&w), "oc_device_status");
  return w;
}

// What a call on t's device needs: its current stream (asked for every time), and the SM count and the status word
// (remembered per device, as they last as long as the process).
Context context_of(const Tensor& t) {
  if (!t.is_cuda()) return {};  // the operator refuses it
  static PyObject* current = nullptr;  // torch._C._cuda_getCurrentRawStream
  static std::vector<std::pair<int64_t, Context>> known;
  if (!current) current = py::object(py::module_::import("torch._C").attr("_cuda_getCurrentRawStream")).release().ptr();
  const int64_t device = t.get_device();
  const py::object handle =
      py::reinterpret_steal<py::object>(PyObject_CallFunction(current, "L", static_cast<long long>(device)));
  if (!handle) throw python_error();
  const int64_t stream = PyLong_AsLongLong(handle.ptr());
  for (const auto& k : known)
    if (k.first == device) return Context{k.second.num_sms, k.second.status, stream};
  const int64_t sms = py::module_::import("orthocache_gpu_b200._lib")
                          .attr("num_sms")(py::reinterpret_steal<py::object>(THPVariable_Wrap(t)).attr("device"))
                          .cast<int64_t>();
  const Context c{sms, reinterpret_cast<int64_t>(status_of(device)), stream};
  known.push_back({device, c});
  return c;
}

const Tensor& tensor(PyObject* o, const char* name) {
  OC_TYPE(THPVariable_Check(o), name, " must be a tensor");
  return THPVariable_Unpack(o);
}
OptTensor maybe(PyObject* o, const char* name) {
  if (o == Py_None) return c10::nullopt;
  return tensor(o, name);
}
double number(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw python_error();
  return x;
}
int64_t whole(PyObject* o) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) throw python_error();
  return x;
}
bool truth(PyObject* o) {
  const int x = PyObject_IsTrue(o);
  if (x < 0) throw python_error();
  return x;
}
PyObject* give(const OptTensor& t) {
  if (t.has_value()) return THPVariable_Wrap(*t);
  Py_RETURN_NONE;
}
PyObject* give(const OptTensor& a, const OptTensor& b) {
  PyObject *x = give(a), *y = give(b);
  PyObject* both = PyTuple_Pack(2, x, y);
  Py_DECREF(x);
  Py_DECREF(y);
  return both;
}

// q, k, v, positions, cos, sin, k_cache, v_cache, tables, seq_ids, interleaved, inverse, k_scale, v_scale, return_keys
PyObject* py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  OC_TYPE(n == 15, "rotary takes 15 arguments");
  const OptTensor q = maybe(a[0], "q"), k = maybe(a[1], "k");
  OC_VALUE(q.has_value() || k.has_value(), "give q, k or both");
  const Context c = context_of(q.has_value() ? *q : *k);
  const bool keys = truth(a[14]);
  const auto r = rotary_append(q, k, maybe(a[2], "v"), tensor(a[3], "positions"), maybe(a[4], "cos"), maybe(a[5], "sin"),
                               maybe(a[6], "k_cache"), maybe(a[7], "v_cache"), maybe(a[8], "block_tables"),
                               maybe(a[9], "seq_ids"), truth(a[10]), truth(a[11]), number(a[12]), number(a[13]), keys,
                               c.num_sms, c.status, c.stream);
  return keys ? give(std::get<0>(r), std::get<1>(r)) : give(std::get<0>(r));
  END_HANDLE_TH_ERRORS
}

// q, k_cache, v_cache, tables, seq_lens, scale or None, softcap, slopes, window, k_scale, v_scale, return_lse
PyObject* py_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  OC_TYPE(n == 12, "decode takes 12 arguments");
  const Tensor& q = tensor(a[0], "q");
  const Context c = context_of(q);
  const double scale = a[5] == Py_None ? 1.0 / std::sqrt((double)(q.dim() ? q.size(-1) : 1)) : number(a[5]);
  const bool lse = truth(a[11]);
  const auto r = paged_decode(q, tensor(a[1], "k_cache"), tensor(a[2], "v_cache"), tensor(a[3], "block_tables"),
                              tensor(a[4], "seq_lens"), scale, number(a[6]), maybe(a[7], "alibi_slopes"), whole(a[8]),
                              number(a[9]), number(a[10]), lse, c.num_sms, c.status, c.stream);
  return lse ? give(std::get<0>(r), std::get<1>(r)) : give(std::get<0>(r));
  END_HANDLE_TH_ERRORS
}

// q, k, v, cu_seqlens, cu_seqlens_k, causal, prefix_lens, window, scale or None, softcap, slopes, return_lse
PyObject* py_prompt(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  OC_TYPE(n == 12, "prompt takes 12 arguments");
  const Tensor& q = tensor(a[0], "q");
  const Context c = context_of(q);
  const double scale = a[8] == Py_None ? 1.0 / std::sqrt((double)(q.dim() ? q.size(-1) : 1)) : number(a[8]);
  const bool lse = truth(a[11]);
  const auto r = prompt(q, tensor(a[1], "k"), tensor(a[2], "v"), maybe(a[3], "cu_seqlens"), maybe(a[4], "cu_seqlens_k"),
                        truth(a[5]), maybe(a[6], "prefix_lens"), whole(a[7]), scale, number(a[9]),
                        maybe(a[10], "alibi_slopes"), lse, c.num_sms, c.status, c.stream);
  return lse ? give(std::get<0>(r), std::get<1>(r)) : give(std::get<0>(r));
  END_HANDLE_TH_ERRORS
}

// caches, src, dst
PyObject* py_copy_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  OC_TYPE(n == 3, "copy_pages takes 3 arguments");
  const Tensor& src = tensor(a[1], "src");
  const Context c = context_of(src);
  copy_pages(a[0], src, tensor(a[2], "dst"), c.num_sms, c.status, c.stream);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// tables, lens, refs, source, block_size
PyObject* py_fork(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  OC_TYPE(n == 5, "fork_sequences takes 5 arguments");
  const Tensor& table = tensor(a[0], "block_tables");
  const Context c = context_of(table);
  const auto r = fork_sequences(table, tensor(a[1], "seq_lens"), tensor(a[2], "refcounts"), tensor(a[3], "source"),
                                whole(a[4]), c.status, c.stream);
  PyObject *x = THPVariable_Wrap(std::get<0>(r)), *y = THPVariable_Wrap(std::get<1>(r)),
           *z = THPVariable_Wrap(std::get<2>(r));
  PyObject* all = PyTuple_Pack(3, x, y, z);
  Py_DECREF(x);
  Py_DECREF(y);
  Py_DECREF(z);
  return all;
  END_HANDLE_TH_ERRORS
}

// caches, tables, lens, refs, wanted, block_size, return_done
PyObject* py_reserve(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  OC_TYPE(n == 7, "reserve_pages takes 7 arguments");
  const Tensor& table = tensor(a[1], "block_tables");
  const Context c = context_of(table);
  return give(reserve_pages(a[0], table, tensor(a[2], "seq_lens"), tensor(a[3], "refcounts"), tensor(a[4], "wanted"),
                            whole(a[5]), truth(a[6]), c.num_sms, c.status, c.stream));
  END_HANDLE_TH_ERRORS
}

// caches, tables, refs
PyObject* py_compact(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  OC_TYPE(n == 3, "compact_pages takes 3 arguments");
  const Tensor& table = tensor(a[1], "block_tables");
  const Context c = context_of(table);
  const auto r = compact_pages(a[0], table, tensor(a[2], "refcounts"), c.num_sms, c.status, c.stream);
  return give(std::get<0>(r), std::get<1>(r));
  END_HANDLE_TH_ERRORS
}

#define OC_METHOD(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr}
PyMethodDef serving_methods[] = {OC_METHOD("rotary", py_rotary), OC_METHOD("decode", py_decode),
                                 OC_METHOD("prompt", py_prompt), OC_METHOD("copy_pages", py_copy_pages),
                                 OC_METHOD("fork_sequences", py_fork), OC_METHOD("reserve_pages", py_reserve),
                                 OC_METHOD("compact_pages", py_compact), {nullptr, nullptr, 0, nullptr}};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "compiled binding of the V2 / V3 decode calls and the paged-serving operators of liborthocache_b200";
  m.def("v2", &v2);
  m.def("v3", &v3);
  m.def("status_word", [](int64_t device) {  // a view of the device's status word
    return at::from_blob(status_of(device), {1},
                         at::TensorOptions().dtype(at::kInt).device(at::Device(at::kCUDA, static_cast<at::DeviceIndex>(device))));
  });
  if (PyModule_AddFunctions(m.ptr(), serving_methods) != 0) throw py::error_already_set();
}
