// C ABI of the sampling operator (declarations and contract in include/mlq.h):
// argument checks and the launch.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "kernels/launch.h"
#include "kernels/sampling.h"
#include "mlq.h"

using namespace mlq;

namespace {

// Weights are summed in units of 2^-44: so many of them stay within 64 bits.
constexpr int kMaxVocab = 1 << 19;
constexpr int kMaxRows = 1 << 20;

int check_sizes(int rows, int vocab) {
  if (rows < 0 || vocab <= 0) return MLQ_ERR_SHAPE;
  return rows > kMaxRows || vocab > kMaxVocab ? MLQ_ERR_UNSUPPORTED : MLQ_OK;
}

}  // namespace

extern "C" {

int mlq_sample_workspace(int rows, int vocab, size_t* bytes) {
  if (bytes == nullptr) return MLQ_ERR_INVALID_ARG;
  const int rc = check_sizes(rows, vocab);
  if (rc != MLQ_OK) return rc;
  *bytes = sample_workspace(rows, vocab);
  return MLQ_OK;
}

int mlq_sample(const mlq_sampling* s, int rows, int vocab, const float* logits, int64_t stride,
               const float* uniform, int32_t* tokens, void* ws, size_t ws_bytes,
               mlq_stream_t stream) {
  const int rc = check_sizes(rows, vocab);
  if (rc != MLQ_OK) return rc;
  if (logits == nullptr || uniform == nullptr || tokens == nullptr || ((uintptr_t)ws & 255u) != 0)
    return MLQ_ERR_INVALID_ARG;
  if (stride < 0) return MLQ_ERR_SHAPE;
  const size_t need = sample_workspace(rows, vocab);
  if (ws_bytes < need || (need > 0 && ws == nullptr)) return MLQ_ERR_BUFFER_TOO_SMALL;
  if (rows == 0) return MLQ_OK;
  const mlq_sampling none = {};
  const mlq_sampling& r = s != nullptr ? *s : none;
  SampleArgs a = {};
  a.rows = rows;
  a.vocab = vocab;
  a.logits = logits;
  a.stride = stride;
  a.uniform = uniform;
  a.temperature = r.temperature;
  a.top_k = r.top_k;
  a.top_p = r.top_p;
  a.min_p = r.min_p;
  a.tokens = tokens;
  return record_hip(launch_sample(a, ws, (hipStream_t)stream));
}

}  // extern "C"
