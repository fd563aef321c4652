// The attention block's operators (include/nemo.h): rotary positions, alone or
// behind a norm of each head, the residual RMSNorm with 8-bit output, products
// of such rows, attention with a sliding window and sinks, and a paged cache
// of 4-bit floats with attention over it. Host-side launch helpers; arguments are checked by the C ABI.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/nemo.h"
#include "nemo_common.h"

namespace nemo {

typedef __bf16 bf16_t;

// Angles of a rotation: pair i turns by turns[i] whole turns a position.
struct RopeAngles {
  const double* turns;  // device [rotary / 2]
  float magnitude;
  int head_dim, rotary;
  bool half;
};
hipError_t launch_rope_apply(const RopeAngles& angles, int type, const nemo_rope_heads& q, const nemo_rope_heads* k,
                             int64_t rows, const int64_t* positions, int64_t base, hipStream_t stream);

hipError_t launch_rope_norm(const RopeAngles& angles, int type, const nemo_rope_heads& q, const nemo_rope_heads* k,
                            const nemo_head_norm& norm, int64_t rows, const int64_t* positions, int64_t base,
                            hipStream_t stream);

hipError_t launch_norm8(const nemo_norm_args& args, hipStream_t stream);

// Bounds of a window as the kernels take them: unbounded sides and larger
// bounds are kUnbounded, which no sum of a position and a bound overflows.
constexpr int kUnbounded = 1 << 30;
// Bytes of workspace with which the keys of a batch's queries are split.
size_t window_workspace(const nemo_attention_config& c, int count, int64_t q_rows, int64_t max_kv);
// The index arrays of requests that follow each other, and each row's position.
hipError_t launch_ragged_index(const Ragged& rows, int64_t* positions, int32_t* q_start, int64_t* kv_start,
                               int32_t* kv_len, hipStream_t stream);
hipError_t launch_window_attention(const nemo_attention_config& c, const nemo_attention_batch& b, hipStream_t stream);

hipError_t launch_matmul8(const nemo_matmul8_args& args, hipStream_t stream);

// Rows into a cache, keys turned by `angles` unless it is null, and out of it.
hipError_t launch_cache4_append(const nemo_cache4_config& c, const nemo_cache4_pages& p, const nemo_cache4_rows& r,
                                const RopeAngles* angles, hipStream_t stream);
hipError_t launch_cache4_read(const nemo_cache4_config& c, const nemo_cache4_pages& p, const nemo_cache4_rows& r,
                              hipStream_t stream);
size_t cache4_workspace(const nemo_attention_config& c, int count, int64_t q_rows, int64_t max_kv);
hipError_t launch_cache4_attention(const nemo_cache4_config& cache, const nemo_attention_config& c,
                                   const nemo_cache4_pages& p, const nemo_cache4_queries& q, hipStream_t stream);

}  // namespace nemo
