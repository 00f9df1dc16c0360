// C ABI of the paged-cache operators (declarations and contracts in
// include/mlq.h): argument checks, the host-side frequency table, and the
// launches. Everything that is on the device is checked by the kernels.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "kernels/launch.h"
#include "kernels/paged.h"
#include "mlq.h"

using namespace mlq;

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// Of a sequence: the kernels count positions, padded to whole tiles, in 32 bits.
constexpr int64_t kMaxTokens = (int64_t)1 << 30;
// A launch holds fewer than 2^32 threads, 2^24 workgroups of 256; with so many
// heads those of a decode launch's sequences stay below that.
constexpr int kMaxHeads = 2048;
constexpr int64_t kMaxGroups = ((int64_t)1 << 24) - 1;

size_t kv_bytes(int type) { return type == MLQ_KV_F32 ? 4 : 2; }

int page_shift_of(int page_size) {
  for (int s = 4; s <= 12; ++s)
    if (page_size == 1 << s) return s;
  return -1;
}

// Everything but the pointers.
int check_geometry(const mlq_paged_cache* c) {
  if (c == nullptr) return MLQ_ERR_INVALID_ARG;
  if (c->type != MLQ_KV_F32 && c->type != MLQ_KV_F16 && c->type != MLQ_KV_BF16)
    return MLQ_ERR_INVALID_ARG;
  if (c->n_layers <= 0 || c->n_pages <= 0 || c->page_size <= 0 || c->n_kv_heads <= 0 ||
      c->head_dim <= 0)
    return MLQ_ERR_SHAPE;
  if (page_shift_of(c->page_size) < 0 || c->head_dim % 8 != 0 || c->head_dim > 256)
    return MLQ_ERR_UNSUPPORTED;
  return MLQ_OK;
}

int check_paged_cache(const mlq_paged_cache* c) {
  const int rc = check_geometry(c);
  if (rc != MLQ_OK) return rc;
  if (c->keys == nullptr || c->values == nullptr || !aligned16(c->keys) || !aligned16(c->values))
    return MLQ_ERR_INVALID_ARG;
  return MLQ_OK;
}

// Bytes of one layer of one of the arrays.
size_t layer_bytes(const mlq_paged_cache* c) {
  return (size_t)c->n_pages * c->n_kv_heads * c->page_size * c->head_dim * kv_bytes(c->type);
}

// A row array of `heads` heads: 16-byte aligned rows that do not overlap.
int check_rows(const void* p, int64_t stride, int64_t floats) {
  if (p == nullptr || !aligned16(p) || stride % 4 != 0) return MLQ_ERR_INVALID_ARG;
  return stride < floats ? MLQ_ERR_SHAPE : MLQ_OK;
}

int check_attention(const mlq_paged_cache* c, int layer, const mlq_paged_batch* b,
                    const mlq_attention_rule* rule, int n_heads, const float* q,
                    int64_t q_stride, const float* out, int64_t out_stride, PagedAttnArgs* a) {
  int rc = check_paged_cache(c);
  if (rc != MLQ_OK) return rc;
  if (b == nullptr || b->block_table == nullptr || b->lengths == nullptr)
    return MLQ_ERR_INVALID_ARG;
  if (b->n_seqs <= 0 || b->max_pages <= 0 || n_heads <= 0 || n_heads % c->n_kv_heads != 0)
    return MLQ_ERR_SHAPE;
  if (layer < 0 || layer >= c->n_layers) return MLQ_ERR_SHAPE;
  if ((int64_t)b->max_pages * c->page_size > kMaxTokens || n_heads > kMaxHeads)
    return MLQ_ERR_UNSUPPORTED;
  const int64_t floats = (int64_t)n_heads * c->head_dim;
  if ((rc = check_rows(q, q_stride, floats)) != MLQ_OK) return rc;
  if ((rc = check_rows(out, out_stride, floats)) != MLQ_OK) return rc;
  mlq_attention_rule none = {};
  const mlq_attention_rule& r = rule != nullptr ? *rule : none;
  if (!std::isfinite(r.scale) || !std::isfinite(r.softcap) || r.softcap < 0.0f || r.window < 0)
    return MLQ_ERR_INVALID_ARG;
  const float scale = r.scale != 0.0f ? r.scale : sqrtf(1.0f / (float)c->head_dim);
  // (scores are multiplied by this, and 0 * inf is not 0)
  if (r.softcap > 0.0f && !std::isfinite(scale / r.softcap)) return MLQ_ERR_INVALID_ARG;
  *a = {};
  a->keys = (const char*)c->keys + layer * layer_bytes(c);
  a->values = (const char*)c->values + layer * layer_bytes(c);
  a->type = c->type;
  a->n_pages = c->n_pages;
  a->page_shift = page_shift_of(c->page_size);
  a->n_kv = c->n_kv_heads;
  a->hd = c->head_dim;
  a->group = n_heads / c->n_kv_heads;
  a->n_seqs = b->n_seqs;
  a->max_pages = b->max_pages;
  a->max_rows = b->max_rows;
  a->block_table = b->block_table;
  a->lengths = b->lengths;
  a->row_start = b->row_start;
  a->q = q;
  a->out = out != nullptr ? const_cast<float*>(out) : nullptr;
  a->q_stride = q_stride;
  a->out_stride = out_stride;
  a->scale = scale;
  a->softcap = r.softcap;
  a->window = r.window;
  a->slopes = r.slopes;
  return MLQ_OK;
}

// A window that every sequence fits in is none (and positions minus a window
// stay within 32 bits).
void bound_lengths(PagedAttnArgs* a, int max_len) {
  a->max_len = max_len;
  if (a->window >= max_len) a->window = 0;
}

}  // namespace

extern "C" {

int mlq_paged_cache_bytes(const mlq_paged_cache* c, size_t* bytes) {
  const int rc = check_geometry(c);
  if (rc != MLQ_OK) return rc;
  if (bytes == nullptr) return MLQ_ERR_INVALID_ARG;
  *bytes = layer_bytes(c) * c->n_layers;
  return MLQ_OK;
}

int mlq_paged_plan(const mlq_paged_batch* b, int page_size, int n_pages, const int32_t* lengths,
                   const int32_t* n_new, int32_t* free_pages, const int32_t* n_free,
                   int32_t* n_free_out, mlq_stream_t stream) {
  if (b == nullptr || b->block_table == nullptr || b->lengths == nullptr ||
      b->row_start == nullptr || b->positions == nullptr || b->slots == nullptr ||
      b->status == nullptr || lengths == nullptr || n_new == nullptr || free_pages == nullptr ||
      n_free == nullptr || n_free_out == nullptr)
    return MLQ_ERR_INVALID_ARG;
  if (b->n_seqs <= 0 || b->max_pages <= 0 || b->max_rows <= 0 || n_pages <= 0 || page_size <= 0)
    return MLQ_ERR_SHAPE;
  const int shift = page_shift_of(page_size);
  if (shift < 0 || (int64_t)b->max_pages * page_size > kMaxTokens) return MLQ_ERR_UNSUPPORTED;
  PlanArgs a = {};
  a.n_seqs = b->n_seqs;
  a.max_pages = b->max_pages;
  a.max_rows = b->max_rows;
  a.page_shift = shift;
  a.n_pages = n_pages;
  a.lengths = lengths;
  a.n_new = n_new;
  a.n_free = n_free;
  a.free_pages = free_pages;
  a.n_free_out = n_free_out;
  a.block_table = b->block_table;
  a.lengths_out = b->lengths;
  a.row_start = b->row_start;
  a.positions = b->positions;
  a.slots = b->slots;
  a.status = b->status;
  return record_hip(launch_paged_plan(a, (hipStream_t)stream));
}

int mlq_rope_frequencies(double theta, int rot_dim, int scaling, double factor, int original_len,
                         double beta_fast, double beta_slow, double* freqs, float* magnitude) {
  if (freqs == nullptr || magnitude == nullptr) return MLQ_ERR_INVALID_ARG;
  if (rot_dim <= 0 || rot_dim % 2 != 0) return MLQ_ERR_SHAPE;
  if (!(std::isfinite(theta) && theta > 0.0)) return MLQ_ERR_INVALID_ARG;
  if (scaling != MLQ_ROPE_SCALE_NONE && scaling != MLQ_ROPE_SCALE_LINEAR &&
      scaling != MLQ_ROPE_SCALE_PARTS)
    return MLQ_ERR_INVALID_ARG;
  if (scaling != MLQ_ROPE_SCALE_NONE && !(std::isfinite(factor) && factor >= 1.0))
    return MLQ_ERR_INVALID_ARG;
  const int half = rot_dim / 2;
  double low = 0.0, high = 0.0;  // pairs below low keep f, above high get f / factor
  if (scaling == MLQ_ROPE_SCALE_PARTS) {
    // (theta = 1 turns every pair alike: no index has a given count of turns)
    if (original_len <= 0 || !(theta > 1.0) || !(std::isfinite(beta_fast) && beta_slow > 0.0 &&
                                                 beta_fast > beta_slow))
      return MLQ_ERR_INVALID_ARG;
    // the pair that turns n times: original_len theta^(-2i/rot) = 2 pi n
    auto index = [&](double n) {
      return rot_dim * std::log(original_len / (2.0 * M_PI * n)) / (2.0 * std::log(theta));
    };
    low = std::fmax(std::floor(index(beta_fast)), 0.0);
    high = std::fmin(std::ceil(index(beta_slow)), rot_dim - 1.0);
    if (!(high > low)) high = low + 0.001;
  }
  for (int i = 0; i < half; ++i) {
    const double f = std::pow(theta, -2.0 * i / rot_dim);
    double slow = scaling == MLQ_ROPE_SCALE_LINEAR ? 1.0 : 0.0;  // share of f / factor
    if (scaling == MLQ_ROPE_SCALE_PARTS)
      slow = std::fmin(std::fmax((i - low) / (high - low), 0.0), 1.0);
    freqs[i] = scaling == MLQ_ROPE_SCALE_NONE ? f : f * (1.0 - slow) + f / factor * slow;
  }
  *magnitude = scaling == MLQ_ROPE_SCALE_PARTS ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
  return MLQ_OK;
}

int mlq_qk_norm_rope(const mlq_rotary* r, int rows, const int32_t* positions, int n_heads,
                     int n_kv_heads, const float* q, int64_t q_stride, const float* k,
                     int64_t k_stride, const float* v, int64_t v_stride, float* q_out,
                     int64_t q_out_stride, float* k_out, int64_t k_out_stride,
                     const mlq_paged_cache* c, int layer, const int64_t* slots,
                     mlq_stream_t stream) {
  if (r == nullptr || positions == nullptr) return MLQ_ERR_INVALID_ARG;
  if (rows < 0 || n_heads <= 0 || n_kv_heads <= 0 || r->head_dim <= 0 || r->rot_dim < 0 ||
      r->rot_dim % 2 != 0 || r->rot_dim > r->head_dim)
    return MLQ_ERR_SHAPE;
  if (r->head_dim % 8 != 0 || r->head_dim > 256 || n_heads > kMaxHeads || n_kv_heads > kMaxHeads ||
      rows > kMaxGroups)
    return MLQ_ERR_UNSUPPORTED;
  if (r->rope_type != MLQ_ROPE_NORMAL && r->rope_type != MLQ_ROPE_NEOX)
    return MLQ_ERR_INVALID_ARG;
  if (r->rot_dim > 0 && (r->freqs == nullptr || !std::isfinite(r->magnitude)))
    return MLQ_ERR_INVALID_ARG;
  if ((r->q_norm != nullptr || r->k_norm != nullptr) && !(std::isfinite(r->eps) && r->eps > 0.0f))
    return MLQ_ERR_INVALID_ARG;
  if (!aligned16(r->q_norm) || !aligned16(r->k_norm)) return MLQ_ERR_INVALID_ARG;
  const int64_t qd = (int64_t)n_heads * r->head_dim, kvd = (int64_t)n_kv_heads * r->head_dim;
  int rc;
  if ((rc = check_rows(q, q_stride, qd)) != MLQ_OK) return rc;
  if ((rc = check_rows(k, k_stride, kvd)) != MLQ_OK) return rc;
  if ((rc = check_rows(q_out, q_out_stride, qd)) != MLQ_OK) return rc;
  if (q_out == q && q_out_stride != q_stride) return MLQ_ERR_INVALID_ARG;
  if (k_out != nullptr) {
    if ((rc = check_rows(k_out, k_out_stride, kvd)) != MLQ_OK) return rc;
    if (k_out == k && k_out_stride != k_stride) return MLQ_ERR_INVALID_ARG;
  }
  RotaryArgs a = {};
  if (c != nullptr) {
    if ((rc = check_paged_cache(c)) != MLQ_OK) return rc;
    if (c->n_kv_heads != n_kv_heads || c->head_dim != r->head_dim || layer < 0 ||
        layer >= c->n_layers)
      return MLQ_ERR_SHAPE;
    if (slots == nullptr) return MLQ_ERR_INVALID_ARG;
    if ((rc = check_rows(v, v_stride, kvd)) != MLQ_OK) return rc;
    a.keys = (char*)c->keys + layer * layer_bytes(c);
    a.values = (char*)c->values + layer * layer_bytes(c);
    a.type = c->type;
    a.page_shift = page_shift_of(c->page_size);
    a.n_slots = (int64_t)c->n_pages * c->page_size;
    a.slots = slots;
    a.v = v;
    a.v_stride = v_stride;
  } else if (k_out == nullptr) {
    return MLQ_ERR_INVALID_ARG;
  }
  if (rows == 0) return MLQ_OK;
  a.rows = rows;
  a.n_heads = n_heads;
  a.n_kv = n_kv_heads;
  a.hd = r->head_dim;
  a.rot = r->rot_dim;
  a.neox = r->rope_type == MLQ_ROPE_NEOX;
  a.magnitude = r->magnitude;
  a.eps = r->eps;
  a.freqs = r->freqs;
  a.q_norm = r->q_norm;
  a.k_norm = r->k_norm;
  a.positions = positions;
  a.q = q;
  a.k = k;
  a.q_out = q_out;
  a.k_out = k_out;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.q_out_stride = q_out_stride;
  a.k_out_stride = k_out_stride;
  return record_hip(launch_qk_norm_rope(a, (hipStream_t)stream));
}

int mlq_paged_attention_workspace(const mlq_paged_cache* c, int n_heads, int n_seqs, int max_rows,
                                  int max_len, size_t* bytes) {
  const int rc = check_geometry(c);
  if (rc != MLQ_OK) return rc;
  if (bytes == nullptr) return MLQ_ERR_INVALID_ARG;
  if (n_heads <= 0 || n_heads % c->n_kv_heads != 0 || n_seqs <= 0 || max_rows < 0 || max_len <= 0)
    return MLQ_ERR_SHAPE;
  if (max_len > kMaxTokens || n_heads > kMaxHeads) return MLQ_ERR_UNSUPPORTED;
  PagedAttnArgs a = {};
  a.type = c->type;
  a.n_kv = c->n_kv_heads;
  a.hd = c->head_dim;
  a.group = n_heads / c->n_kv_heads;
  a.n_seqs = n_seqs;
  a.max_len = max_len;
  a.max_rows = max_rows;
  if (max_rows > 0 && prefill_groups(a) > kMaxGroups) return MLQ_ERR_UNSUPPORTED;
  *bytes = max_rows == 0 ? plan_paged_decode(a) : plan_paged_prefill(a);
  return MLQ_OK;
}

int mlq_paged_attention_decode(const mlq_paged_cache* c, int layer, const mlq_paged_batch* b,
                               const mlq_attention_rule* rule, int n_heads, const float* q,
                               int64_t q_stride, float* out, int64_t out_stride, int max_len,
                               void* ws, size_t ws_bytes, mlq_stream_t stream) {
  PagedAttnArgs a;
  const int rc = check_attention(c, layer, b, rule, n_heads, q, q_stride, out, out_stride, &a);
  if (rc != MLQ_OK) return rc;
  if (max_len <= 0 || max_len > (int64_t)b->max_pages * c->page_size) return MLQ_ERR_SHAPE;
  if (b->row_start == nullptr)
    a.max_rows = b->n_seqs;
  else if (b->max_rows <= 0)
    return MLQ_ERR_SHAPE;
  bound_lengths(&a, max_len);
  const size_t need = plan_paged_decode(a);
  if (((uintptr_t)ws & 255u) != 0) return MLQ_ERR_INVALID_ARG;
  if (ws_bytes < need || (need > 0 && ws == nullptr)) return MLQ_ERR_BUFFER_TOO_SMALL;
  if (out == q) return MLQ_ERR_INVALID_ARG;  // (q is read again after some of out is written)
  a.part = need > 0 ? ws : nullptr;
  return record_hip(launch_paged_decode(a, (hipStream_t)stream));
}

int mlq_paged_attention_prefill(const mlq_paged_cache* c, int layer, const mlq_paged_batch* b,
                                const mlq_attention_rule* rule, int n_heads, const float* q,
                                int64_t q_stride, float* out, int64_t out_stride, int max_len,
                                void* ws, size_t ws_bytes, mlq_stream_t stream) {
  PagedAttnArgs a;
  const int rc = check_attention(c, layer, b, rule, n_heads, q, q_stride, out, out_stride, &a);
  if (rc != MLQ_OK) return rc;
  if (b->row_start == nullptr) return MLQ_ERR_INVALID_ARG;
  if (b->max_rows <= 0 || max_len <= 0 || max_len > (int64_t)b->max_pages * c->page_size)
    return MLQ_ERR_SHAPE;
  bound_lengths(&a, max_len);
  if (prefill_groups(a) > kMaxGroups) return MLQ_ERR_UNSUPPORTED;
  const size_t need = plan_paged_prefill(a);
  if (((uintptr_t)ws & 255u) != 0) return MLQ_ERR_INVALID_ARG;
  if (ws_bytes < need || (need > 0 && ws == nullptr)) return MLQ_ERR_BUFFER_TOO_SMALL;
  if (out == q) return MLQ_ERR_INVALID_ARG;  // (q is read again after some of out is written)
  a.part = need > 0 ? ws : nullptr;
  return record_hip(launch_paged_prefill(a, (hipStream_t)stream));
}

}  // extern "C"
