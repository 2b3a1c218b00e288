// ragged_abi.cu — entry points of the ragged-batch operators: argument checks
// and the launch structures of kv_append.cu and attention_ragged.cu.
//
// Nothing here keeps state or allocates: every call is one kernel on the
// caller's stream that touches only the caller's buffers and the engine's error
// word, so calls may run at the same time on any streams and inside graphs.
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "kernels.h"

using namespace rb;

namespace {

int refuse(int rc, const char* fmt, ...) {
  char msg[320];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  return report_error(rc, msg);
}

constexpr int64_t kMaxRows = int64_t(1) << 30;

struct Heads {
  int n_head, n_kv_heads, d;
};

int check_common(const char* op, int dtype, int64_t tokens, int64_t batch, const Heads& h) {
  if (dtype != RB_DTYPE_F16 && dtype != RB_DTYPE_BF16)
    return refuse(RB_E_SHAPE, "%s: dtype %d (f16 and bf16 only)", op, dtype);
  if (tokens < 0 || tokens > kMaxRows || batch < 0 || batch > kMaxRows)
    return refuse(RB_E_SHAPE, "%s: tokens=%lld batch=%lld", op, (long long)tokens, (long long)batch);
  if (h.n_head <= 0 || h.n_kv_heads <= 0 || h.n_head % h.n_kv_heads != 0 || h.n_head / h.n_kv_heads > 128 ||
      h.n_head > 65535)
    return refuse(RB_E_SHAPE, "%s: n_head=%d n_kv_heads=%d (a multiple, at most 128 query heads a KV head)", op,
                  h.n_head, h.n_kv_heads);
  return RB_OK;
}

// Rows of `heads` heads that start on 16-byte boundaries.
int check_rows(const char* op, const char* what, const void* p, int64_t ld, int heads, int d) {
  if (!p) return refuse(RB_E_SHAPE, "%s: null %s", op, what);
  if (ld < static_cast<int64_t>(heads) * d || ld > (int64_t(1) << 31))
    return refuse(RB_E_SHAPE, "%s: %s row stride %lld below heads * head_dim = %lld", op, what, (long long)ld,
                  (long long)heads * d);
  if ((reinterpret_cast<uintptr_t>(p) & 15) != 0 || ld % 8 != 0)
    return refuse(RB_E_SHAPE, "%s: %s rows must start on 16-byte boundaries", op, what);
  return RB_OK;
}

// (`empty`: a call without tokens or sequences, whose table may have no address.)
int check_cache(const char* op, const Heads& h, const void* k, const void* v, int64_t page_stride, int64_t num_pages,
                int page_size, const int32_t* table, int64_t ld_table, bool empty, KeyValues* kv) {
  if (h.d != 64 && h.d != 128)
    return refuse(RB_E_UNSUPPORTED, "%s: head_dim %d (supported: 64, 128)", op, h.d);
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
    return refuse(RB_E_UNSUPPORTED, "%s: page_size %d (supported: 16, 32, 64, 128)", op, page_size);
  if (num_pages <= 0 || num_pages > kMaxRows || (!empty && (ld_table <= 0 || !table)))
    return refuse(RB_E_SHAPE, "%s: num_pages=%lld, page table width %lld", op, (long long)num_pages,
                  (long long)ld_table);
  const int64_t row = static_cast<int64_t>(h.n_kv_heads) * h.d;
  if (page_stride < row * page_size || page_stride % 8 != 0 || page_stride > (int64_t(1) << 38))
    return refuse(RB_E_SHAPE, "%s: page stride %lld elements (at least %lld, a multiple of 8)", op,
                  (long long)page_stride, (long long)(row * page_size));
  int rc;
  if ((rc = check_rows(op, "k_cache", k, row, h.n_kv_heads, h.d)) != RB_OK ||
      (rc = check_rows(op, "v_cache", v, row, h.n_kv_heads, h.d)) != RB_OK)
    return rc;
  kv->k = static_cast<const uint16_t*>(k);
  kv->v = static_cast<const uint16_t*>(v);
  kv->ldk = kv->ldv = row;
  kv->table = table;
  kv->ld_table = ld_table;
  kv->page_stride = page_stride;
  kv->page_shift = page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : 7;
  kv->num_pages = static_cast<int>(num_pages);
  return RB_OK;
}

int check_softmax(const char* op, float scale, float softcap) {
  if (!(scale > 0.0f) || std::isinf(scale) || !(softcap >= 0.0f) || std::isinf(softcap))
    return refuse(RB_E_SHAPE, "%s: scale %g must be positive and softcap %g zero (none) or positive", op,
                  static_cast<double>(scale), static_cast<double>(softcap));
  return RB_OK;
}

int band(int64_t window) {  // window >= 0 as a band bound
  return static_cast<int>(window > kRaggedNoBound / 2 ? kRaggedNoBound / 2 : window);
}

int most_keys(int64_t ld_table, int page_size) {
  return static_cast<int>(ld_table > kMaxRows / page_size ? kMaxRows : ld_table * page_size);
}

}  // namespace

extern "C" int rb_kv_append(const rb_kv_append_args* args, void* stream) {
  if (!args) return report_error(RB_E_SHAPE, "kv_append: null arguments");
  const auto [q, k, v, ldq, ldk, ldv, tokens, batch, cu_q, kv_len, q_norm_w, k_norm_w, cos_t, sin_t, max_pos, q_out,
              ldq_out, k_cache, v_cache, page_stride, num_pages, page_table, ld_table, dtype, n_head, n_kv_heads,
              head_dim, page_size, eps] = *args;
  const char* op = "kv_append";
  int rc;
  const Heads h{n_head, n_kv_heads, head_dim};
  KvAppend a{};
  if ((rc = check_common(op, dtype, tokens, batch, h)) != RB_OK ||
      (rc = check_cache(op, h, k_cache, v_cache, page_stride, num_pages, page_size, page_table, ld_table,
                        tokens == 0 || batch == 0, &a.cache)) != RB_OK)
    return rc;
  if (!(eps >= 0.0f)) return refuse(RB_E_SHAPE, "%s: eps %g", op, static_cast<double>(eps));
  if (tokens == 0 || batch == 0) return RB_OK;
  if ((rc = check_rows(op, "q", q, ldq, n_head, head_dim)) != RB_OK ||
      (rc = check_rows(op, "k", k, ldk, n_kv_heads, head_dim)) != RB_OK ||
      (rc = check_rows(op, "v", v, ldv, n_kv_heads, head_dim)) != RB_OK ||
      (rc = check_rows(op, "q_out", q_out, ldq_out, n_head, head_dim)) != RB_OK)
    return rc;
  if (q_out == k || q_out == v || q_out == k_cache || q_out == v_cache)
    return refuse(RB_E_SHAPE, "%s: q_out may be q, but no other input", op);
  if (q_out == q && ldq_out != ldq) return refuse(RB_E_SHAPE, "%s: q in place needs one row stride", op);
  if (!cu_q || !kv_len || !cos_t || !sin_t || max_pos <= 0 || max_pos > kMaxRows)
    return refuse(RB_E_SHAPE, "%s: null cu_q, kv_len, cos or sin, or max_pos=%lld", op, (long long)max_pos);
  for (const float* p : {q_norm_w, k_norm_w, cos_t, sin_t})
    if ((reinterpret_cast<uintptr_t>(p) & 15) != 0)
      return refuse(RB_E_SHAPE, "%s: norm weights, cos and sin must be 16-byte aligned", op);
  EngineView e;
  if ((rc = engine_view(&e)) != RB_OK) return rc;
  a.seqs = {cu_q, kv_len, static_cast<int>(batch), static_cast<int>(tokens), static_cast<int>(tokens),
            most_keys(ld_table, page_size), e.err};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.ldq = ldq;
  a.ldk = ldk;
  a.ldv = ldv;
  a.ldo = ldq_out;
  a.n_head = n_head;
  a.n_kv_heads = n_kv_heads;
  a.head_dim = head_dim;
  a.bf16 = dtype == RB_DTYPE_BF16;
  a.q_norm = q_norm_w;
  a.k_norm = k_norm_w;
  a.eps = eps;
  a.cos_t = cos_t;
  a.sin_t = sin_t;
  a.max_pos = static_cast<int>(max_pos);
  a.q_out = static_cast<uint16_t*>(q_out);
  a.k_cache = static_cast<uint16_t*>(k_cache);
  a.v_cache = static_cast<uint16_t*>(v_cache);
  if ((rc = launch_kv_append(a, static_cast<cudaStream_t>(stream))) != RB_OK) return rc;
  count_launches(1);
  return RB_OK;
}

extern "C" int rb_attention_paged(const rb_attention_paged_args* args, void* stream) {
  if (!args) return report_error(RB_E_SHAPE, "attention_paged: null arguments");
  const auto [q, out, k_cache, v_cache, ldq, ldo, tokens, batch, cu_q, kv_len, max_q, max_kv, page_stride, num_pages,
              page_table, ld_table, window, dtype, n_head, n_kv_heads, head_dim, page_size, scale, softcap] = *args;
  const char* op = "attention_paged";
  int rc;
  const Heads h{n_head, n_kv_heads, head_dim};
  AttnRagged a{};
  if ((rc = check_common(op, dtype, tokens, batch, h)) != RB_OK ||
      (rc = check_cache(op, h, k_cache, v_cache, page_stride, num_pages, page_size, page_table, ld_table,
                        tokens == 0 || batch == 0, &a.kv)) != RB_OK ||
      (rc = check_softmax(op, scale, softcap)) != RB_OK)
    return rc;
  if (max_q < 0 || max_kv < 0) return refuse(RB_E_SHAPE, "%s: max_q=%lld max_kv=%lld", op, (long long)max_q, (long long)max_kv);
  if (tokens == 0 || batch == 0) return RB_OK;
  if ((rc = check_rows(op, "q", q, ldq, n_head, head_dim)) != RB_OK ||
      (rc = check_rows(op, "out", out, ldo, n_head, head_dim)) != RB_OK)
    return rc;
  if (out == q || out == k_cache || out == v_cache) return refuse(RB_E_SHAPE, "%s: out must not be an input", op);
  if (!cu_q || !kv_len) return refuse(RB_E_SHAPE, "%s: null cu_q or kv_len", op);
  EngineView e;
  if ((rc = engine_view(&e)) != RB_OK) return rc;
  const int most = most_keys(ld_table, page_size);
  a.seqs = {cu_q, kv_len, static_cast<int>(batch), static_cast<int>(tokens),
            static_cast<int>(max_q < tokens ? max_q : tokens), most, e.err};
  a.hint_kv = static_cast<int>(max_kv > 0 && max_kv < most ? max_kv : most);
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.ldq = ldq;
  a.ldo = ldo;
  a.n_head = n_head;
  a.n_kv_heads = n_kv_heads;
  a.head_dim = head_dim;
  a.bf16 = dtype == RB_DTYPE_BF16;
  a.scale = scale;
  a.softcap = softcap;
  a.dlo = window < 0 ? -kRaggedNoBound : 1 - band(window);
  a.dhi = 0;
  a.num_sms = e.num_sms;
  if ((rc = launch_attention_ragged(a, static_cast<cudaStream_t>(stream))) != RB_OK) return rc;
  count_launches(1);
  return RB_OK;
}

extern "C" int rb_attention_packed(const rb_attention_packed_args* args, void* stream) {
  if (!args) return report_error(RB_E_SHAPE, "attention_packed: null arguments");
  const auto [q, k, v, out, ldq, ldk, ldv, ldo, tokens, batch, cu_seqlens, window, dtype, n_head, n_kv_heads, head_dim,
              mask_mode, scale, softcap] = *args;
  const char* op = "attention_packed";
  int rc;
  const Heads h{n_head, n_kv_heads, head_dim};
  if ((rc = check_common(op, dtype, tokens, batch, h)) != RB_OK || (rc = check_softmax(op, scale, softcap)) != RB_OK)
    return rc;
  if (head_dim != 64 && head_dim != 72 && head_dim != 128)
    return refuse(RB_E_UNSUPPORTED, "%s: head_dim %d (supported: 64, 72, 128)", op, head_dim);
  if (mask_mode != RB_MASK_NONE && mask_mode != RB_MASK_CAUSAL && mask_mode != RB_MASK_WINDOW &&
      mask_mode != RB_MASK_CAUSAL_WINDOW)
    return refuse(RB_E_SHAPE, "%s: mask mode %d (the full-sequence modes only)", op, mask_mode);
  if (tokens == 0 || batch == 0) return RB_OK;
  if ((rc = check_rows(op, "q", q, ldq, n_head, head_dim)) != RB_OK ||
      (rc = check_rows(op, "k", k, ldk, n_kv_heads, head_dim)) != RB_OK ||
      (rc = check_rows(op, "v", v, ldv, n_kv_heads, head_dim)) != RB_OK ||
      (rc = check_rows(op, "out", out, ldo, n_head, head_dim)) != RB_OK)
    return rc;
  if (out == q || out == k || out == v) return refuse(RB_E_SHAPE, "%s: out must not be an input", op);
  if (!cu_seqlens) return refuse(RB_E_SHAPE, "%s: null cu_seqlens", op);
  EngineView e;
  if ((rc = engine_view(&e)) != RB_OK) return rc;
  AttnRagged a{};
  a.seqs = {cu_seqlens, nullptr, static_cast<int>(batch), static_cast<int>(tokens), static_cast<int>(tokens),
            static_cast<int>(tokens), e.err};
  a.hint_kv = static_cast<int>(batch == 1 ? tokens : std::min(tokens, 2 * tokens / batch + 1));  // twice the mean
  a.kv.k = static_cast<const uint16_t*>(k);
  a.kv.v = static_cast<const uint16_t*>(v);
  a.kv.ldk = ldk;
  a.kv.ldv = ldv;
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.ldq = ldq;
  a.ldo = ldo;
  a.n_head = n_head;
  a.n_kv_heads = n_kv_heads;
  a.head_dim = head_dim;
  a.bf16 = dtype == RB_DTYPE_BF16;
  a.scale = scale;
  a.softcap = softcap;
  const bool causal = mask_mode == RB_MASK_CAUSAL || mask_mode == RB_MASK_CAUSAL_WINDOW;
  const bool windowed = (mask_mode == RB_MASK_WINDOW || mask_mode == RB_MASK_CAUSAL_WINDOW) && window >= 0;
  a.dlo = !windowed ? -kRaggedNoBound : causal ? 1 - band(window) : -band(window);
  a.dhi = causal ? 0 : windowed ? band(window) : kRaggedNoBound;
  a.num_sms = e.num_sms;
  if ((rc = launch_attention_ragged(a, static_cast<cudaStream_t>(stream))) != RB_OK) return rc;
  count_launches(1);
  return RB_OK;
}
