// C entries of the q/k norms and the E4M3 paged KV cache (kernels: csrc/qk_norm.cu,
// csrc/kv8.cu): argument checks, then one asynchronous launch (two for the norm's
// gradient) on the caller's stream. No reference counterparts.
#include <climits>
#include <cmath>
#include <cstdio>
#include <exception>

#include "engine.hpp"

namespace wv {

Status kv8_supported(const Cfg& c, const char* who) {
  if (c.c.precision != 1) return Status::err(2, std::string(who) + ": the E4M3 cache needs BF16 activations (precision 1)");
  if (c.c.softmax != 0) return Status::err(2, std::string(who) + ": the E4M3 cache needs softmax scores");
  if (c.c.mask != 1 && !(c.c.mask == 3 && c.c.window_causal))
    return Status::err(2, std::string(who) + ": the E4M3 cache needs the causal or the causal window mask");
  if (c.hd % 2 || c.hd > kKv8MaxHeadDim)
    return Status::err(2, std::string(who) + ": the E4M3 cache needs an even head_dim of at most " + std::to_string(kKv8MaxHeadDim));
  return Status::ok();
}

void kv8_mask(const Cfg& c, Kv8AttnArgs* a) {
  a->window = c.c.mask == 3 ? (c.c.window > 0 ? c.c.window : c.msl) : 0;
  a->alibi = c.alibi;
  a->head_base = c.c.head_begin;
  a->total_heads = c.c.num_heads;
  a->scale = c.scale;
}

namespace {

// Runs a C entry's body; an exception (no memory for a message) becomes code 4.
template <class F> welvet_status entry(const char* name, F&& body) {
  try {
    DeviceRestore restore_device;
    return to_c(body());
  } catch (const std::exception& e) {
    welvet_status st{};
    st.code = 4;
    std::snprintf(st.message, sizeof(st.message), "%s: %s", name, e.what());
    return st;
  }
}

// Whether every pointer (null ones aside) is a multiple of n bytes: kernels load rows by
// element at least, and a table's (cos, sin) together.
template <class... P> bool aligned(size_t n, const P*... p) {
  return ((reinterpret_cast<uintptr_t>(p) % n == 0) && ...);
}

Status norm_args(const char* name, int64_t tokens, int heads, int kv_heads, int head_dim, double eps,
                 const float* q_gamma, const float* k_gamma, const float* rope, int max_pos, const int* positions,
                 int pos_mod, const void* q, int64_t ldq, const void* k, int64_t ldk, void* q_out, int64_t ldqo,
                 void* k_out, int64_t ldko, int io_bf16, QkNormArgs* out) {
  const std::string who(name);
  if (tokens < 0 || heads < 0 || kv_heads < 0 || heads + (int64_t)kv_heads <= 0 || head_dim <= 0 ||
      (rope && max_pos <= 0) || std::isnan(eps))
    return Status::err(1, who + ": invalid argument");
  if (head_dim % 2 || head_dim > kQkNormMaxHeadDim)
    return Status::err(2, who + ": head_dim must be even and at most " + std::to_string(kQkNormMaxHeadDim));
  const int64_t qd = (int64_t)heads * head_dim, kd = (int64_t)kv_heads * head_dim;
  if (tokens > 0 && ((heads && (!q || !q_out)) || (kv_heads && (!k || !k_out))))
    return Status::err(1, who + ": invalid argument");
  if (!aligned(io_bf16 ? 2 : 4, q, k, q_out, k_out) || !aligned(4, q_gamma, k_gamma, positions) || !aligned(8, rope))
    return Status::err(1, who + ": misaligned pointer");
  if ((heads && (ldq < qd || ldqo < qd)) || (kv_heads && (ldk < kd || ldko < kd)))
    return Status::err(1, who + ": row stride smaller than heads * head_dim");
  if (tokens > INT_MAX || tokens * (heads + (int64_t)kv_heads) > INT_MAX)
    return Status::err(1, who + ": tokens * heads too large");
  QkNormArgs& a = *out;
  a.tokens = tokens;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.head_dim = head_dim;
  a.is_bf16 = io_bf16 != 0;
  a.eps = eps > 0 ? (float)eps : 1e-6f;
  a.q_gamma = q_gamma;
  a.k_gamma = k_gamma;
  a.rope = reinterpret_cast<const float2*>(rope);
  a.max_pos = max_pos;
  a.positions = positions;
  a.pos_mod = pos_mod;
  a.q = q;
  a.k = k;
  a.ldq = ldq;
  a.ldk = ldk;
  a.q_out = q_out;
  a.k_out = k_out;
  a.ldqo = ldqo;
  a.ldko = ldko;
  return Status::ok();
}

// The current device's part of the arguments, after the checks that need none.
template <class Args> Status on_device(Args* a) {
  DeviceCtx* d = nullptr;
  WV_TRY(device_ctx(-1, &d));
  a->err = d->err;
  a->sm_count = d->sm_count;
  return Status::ok();
}

Status cache_args(const char* name, const welvet_b200_kv8_cache* c, int seq, Kv8Cache* out) {
  const std::string who(name);
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->block_table || !c->ctx_len || c->batch <= 0 ||
      c->pages <= 0 || c->max_pages <= 0 || c->kv_heads <= 0 || c->head_dim <= 0 || seq <= 0)
    return Status::err(1, who + ": invalid argument");
  if (c->head_dim % 2 || c->head_dim > kKv8MaxHeadDim)
    return Status::err(2, who + ": head_dim must be even and at most " + std::to_string(kKv8MaxHeadDim));
  if (c->batch > 65535 || c->kv_heads > 32767 || c->max_pages > INT_MAX / kKv8Page)
    return Status::err(1, who + ": batch, kv_heads or max_pages too large");
  if (!aligned(4, c->k_scale, c->v_scale, c->block_table, c->ctx_len)) return Status::err(1, who + ": misaligned pointer");
  out->k = c->k;
  out->v = c->v;
  out->k_scale = c->k_scale;
  out->v_scale = c->v_scale;
  out->block_table = c->block_table;
  out->ctx_len = c->ctx_len;
  out->pages = c->pages;
  out->max_pages = c->max_pages;
  out->kv_heads = c->kv_heads;
  out->head_dim = c->head_dim;
  return Status::ok();
}

}  // namespace
}  // namespace wv

extern "C" {

welvet_status welvet_b200_rope_table(int32_t max_pos, int32_t head_dim, double theta, float* table, void* stream) {
  return wv::entry("rope_table", [&]() -> wv::Status {
    if (max_pos <= 0 || head_dim < 2 || head_dim % 2 || !(theta > 0) || !table)
      return wv::Status::err(1, "rope_table: invalid argument");
    if (!wv::aligned(8, table)) return wv::Status::err(1, "rope_table: misaligned pointer");
    wv::DeviceCtx* d = nullptr;
    WV_TRY(wv::device_ctx(-1, &d));
    WV_CUDA(wv::rope_table(reinterpret_cast<float2*>(table), max_pos, head_dim, theta, static_cast<cudaStream_t>(stream)),
            "rope_table");
    wv::count_launch();
    return wv::Status::ok();
  });
}

welvet_status welvet_b200_qk_norm_rope_forward(int64_t tokens, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                               double eps, const float* q_gamma, const float* k_gamma,
                                               const float* rope, int32_t max_pos, const int32_t* positions,
                                               int32_t pos_mod, const void* q, int64_t ldq, const void* k, int64_t ldk,
                                               void* q_out, int64_t ldq_out, void* k_out, int64_t ldk_out,
                                               int32_t io_bf16, void* stream) {
  return wv::entry("qk_norm_rope", [&]() -> wv::Status {
    wv::QkNormArgs a;
    WV_TRY(wv::norm_args("qk_norm_rope", tokens, heads, kv_heads, head_dim, eps, q_gamma, k_gamma, rope, max_pos,
                         positions, pos_mod, q, ldq, k, ldk, q_out, ldq_out, k_out, ldk_out, io_bf16, &a));
    WV_TRY(wv::on_device(&a));
    if (tokens == 0) return wv::Status::ok();
    WV_CUDA(wv::qk_norm_forward(a, static_cast<cudaStream_t>(stream)), "qk_norm_rope");
    wv::count_launch();
    return wv::Status::ok();
  });
}

int64_t welvet_b200_qk_norm_rope_workspace(int32_t head_dim) {
  return head_dim > 0 && head_dim <= wv::kQkNormMaxHeadDim ? (int64_t)wv::qk_norm_workspace_bytes(head_dim) : 0;
}

welvet_status welvet_b200_qk_norm_rope_backward(int64_t tokens, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                                double eps, const float* q_gamma, const float* k_gamma,
                                                const float* rope, int32_t max_pos, const int32_t* positions,
                                                int32_t pos_mod, const void* q, int64_t ldq, const void* k,
                                                int64_t ldk, const void* dq_out, int64_t lddq_out,
                                                const void* dk_out, int64_t lddk_out, void* dq, int64_t lddq, void* dk,
                                                int64_t lddk, float* dq_gamma, float* dk_gamma, void* workspace,
                                                int32_t io_bf16, void* stream) {
  return wv::entry("qk_norm_rope_backward", [&]() -> wv::Status {
    const char* name = "qk_norm_rope_backward";
    wv::QkNormArgs a;
    WV_TRY(wv::norm_args(name, tokens, heads, kv_heads, head_dim, eps, q_gamma, k_gamma, rope, max_pos, positions,
                         pos_mod, q, ldq, k, ldk, dq, lddq, dk, lddk, io_bf16, &a));
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || (tokens > 0 && heads && !dq_out) ||
        (tokens > 0 && kv_heads && !dk_out) || (dq_gamma && !q_gamma) || (dk_gamma && !k_gamma))
      return wv::Status::err(1, std::string(name) + ": invalid argument");
    if (!wv::aligned(io_bf16 ? 2 : 4, dq_out, dk_out) || !wv::aligned(4, dq_gamma, dk_gamma))
      return wv::Status::err(1, std::string(name) + ": misaligned pointer");
    if ((heads && lddq_out < (int64_t)heads * head_dim) || (kv_heads && lddk_out < (int64_t)kv_heads * head_dim))
      return wv::Status::err(1, std::string(name) + ": row stride smaller than heads * head_dim");
    WV_TRY(wv::on_device(&a));
    a.dq_out = dq_out;
    a.dk_out = dk_out;
    a.lddqo = lddq_out;
    a.lddko = lddk_out;
    a.dq_gamma = dq_gamma;
    a.dk_gamma = dk_gamma;
    a.partial = static_cast<float*>(workspace);
    WV_CUDA(wv::qk_norm_backward(a, static_cast<cudaStream_t>(stream)), name);
    wv::count_launch(dq_gamma || dk_gamma ? 2 : 1);
    return wv::Status::ok();
  });
}

welvet_status welvet_b200_kv8_append(const welvet_b200_kv8_cache* cache, int32_t seq, const int32_t* seq_lens,
                                     const void* k, int32_t ldk, const void* v, int32_t ldv, const float* rope,
                                     int32_t max_pos, void* stream) {
  return wv::entry("kv8_append", [&]() -> wv::Status {
    wv::Kv8AppendArgs a;
    WV_TRY(wv::cache_args("kv8_append", cache, seq, &a.c));
    const int64_t row = (int64_t)cache->kv_heads * cache->head_dim;
    if (!k || !v || (rope && max_pos <= 0)) return wv::Status::err(1, "kv8_append: invalid argument");
    if (!wv::aligned(2, k, v) || !wv::aligned(4, seq_lens) || !wv::aligned(8, rope))
      return wv::Status::err(1, "kv8_append: misaligned pointer");
    if (ldk < row || ldv < row) return wv::Status::err(1, "kv8_append: row stride smaller than kv_heads * head_dim");
    WV_TRY(wv::on_device(&a));
    a.batch = cache->batch;
    a.seq = seq;
    a.seq_lens = seq_lens;
    a.k = k;
    a.v = v;
    a.ldk = ldk;
    a.ldv = ldv;
    a.rope = reinterpret_cast<const float2*>(rope);
    a.max_pos = max_pos;
    WV_CUDA(wv::kv8_append(a, static_cast<cudaStream_t>(stream)), "kv8_append");
    wv::count_launch();
    return wv::Status::ok();
  });
}

welvet_status welvet_b200_kv8_attention(const welvet_b200_mha_config* cfg, const welvet_b200_kv8_cache* cache,
                                        int32_t seq, const int32_t* seq_lens, int32_t max_ctx, const void* q,
                                        int32_t ldq, void* out, int32_t ldo, void* stream) {
  return wv::entry("kv8_attention", [&]() -> wv::Status {
    if (!cfg || !q || !out || max_ctx <= 0) return wv::Status::err(1, "kv8_attention: invalid argument");
    wv::Kv8AttnArgs a;
    WV_TRY(wv::cache_args("kv8_attention", cache, seq, &a.c));
    if (!wv::aligned(2, q, out) || !wv::aligned(4, seq_lens)) return wv::Status::err(1, "kv8_attention: misaligned pointer");
    wv::Cfg c;
    WV_TRY(wv::resolve_config(*cfg, &c));
    a.heads = c.c.head_count;
    if (a.heads <= 0 || cache->kv_heads != a.heads / c.group || cache->head_dim != c.hd)
      return wv::Status::err(1, "kv8_attention: the cache's kv_heads or head_dim differ from the configuration's");
    if (ldq < (int64_t)a.heads * c.hd || ldo < (int64_t)a.heads * c.hd)
      return wv::Status::err(1, "kv8_attention: ldq/ldo smaller than heads*head_dim");
    if ((int64_t)seq * a.heads > INT_MAX) return wv::Status::err(1, "kv8_attention: seq * heads too large");
    WV_TRY(wv::kv8_supported(c, "kv8_attention"));
    wv::DeviceCtx* d = nullptr;
    WV_TRY(wv::device_ctx(c.c.device, &d));
    a.batch = cache->batch;
    a.seq = seq;
    a.seq_lens = seq_lens;
    a.max_ctx = max_ctx;
    a.q = q;
    a.out = out;
    a.ldq = ldq;
    a.ldo = ldo;
    wv::kv8_mask(c, &a);
    a.err = d->err;
    a.sm_count = d->sm_count;
    WV_CUDA(wv::kv8_attention(a, static_cast<cudaStream_t>(stream)), "kv8_attention");
    wv::count_launch();
    return wv::Status::ok();
  });
}

}  // extern "C"
