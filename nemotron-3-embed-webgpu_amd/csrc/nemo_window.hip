// Attention with a sliding window and sinks for gfx950 (include/nemo.h
// nemo_window_attention): softmax(scale q.k) v over the keys j <= p + right
// that have j >= p - left or j < sinks.
#include <algorithm>

#include "nemo_operators.h"

namespace nemo {

namespace {

struct WindowArgs {
  nemo_attention_batch b;
  int group, left, right, sinks;
  float scale2;  // of the scores, in units of log2
};

// The keys that a query at p sees of a request's n: [0, sinks) and [lo, hi).
struct Seen {
  int sinks, lo, hi;
  __device__ __forceinline__ Seen(const WindowArgs& a, int p, int n) {
    hi = max(0, min(n, a.right >= kUnbounded ? n : p + a.right + 1));
    lo = a.left >= kUnbounded ? 0 : min(hi, max(0, p - a.left));
    sinks = min(a.sinks, lo);
  }
};

// A request as it lies in the buffers, whatever the index arrays hold.
struct Request {
  int q0, queries, keys;
  int64_t kv0;
  __device__ __forceinline__ Request(const nemo_attention_batch& b, int i) {
    q0 = min(max(b.q_start[i], 0), (int)b.q_rows);
    queries = max(min(b.q_start[i + 1], (int)b.q_rows) - q0, 0);
    kv0 = min(max(b.kv_start[i], (int64_t)0), b.kv_rows);
    keys = (int)min((int64_t)max(b.kv_len[i], 0), b.kv_rows - kv0);
  }
};

// Tiles of `rows` (query, head of the group) rows are numbered through a
// batch without a table: request i's first is floor(q_start[i] group / rows)
// + i, which leaves it at least as many numbers as it has tiles. The request
// of tile number t, -1 if it is none's.
__device__ __forceinline__ int tile_base(const nemo_attention_batch& b, int group, int rows, int i) {
  const int q0 = min(max(b.q_start[i], 0), (int)b.q_rows);
  return (int)((int64_t)q0 * group / rows) + i;
}
__device__ __forceinline__ int tile_request(const nemo_attention_batch& b, int group, int rows, int t) {
  int found = 0;
  for (int i0 = 0; i0 < b.count; i0 += 64) {
    const int i = i0 + (int)(threadIdx.x & 63);
    const uint64_t at = __builtin_amdgcn_ballot_w64(i < b.count && tile_base(b, group, rows, i) <= t);
    found += (int)__popcll(at);
    if (at != ~0ull) break;
  }
  return found - 1;
}

// One query head over keys [j0, j1), by a wave: its running maximum, sum and
// output columns lane, lane + 64.
template <typename T, int HD>
struct OneRow {
  float m = -INFINITY, l = 0.f, o[HD / 64] = {};
  __device__ __forceinline__ void keys(const T* q, const T* k, int64_t k_row, const T* v, int64_t v_row, int j0,
                                       int j1, float scale2) {
    const int lane = threadIdx.x & 63;
    for (int jb = j0; jb < j1; jb += 64) {
      const int j = jb + lane;
      float s = 0.f;
      if (j < j1)
        for (int d = 0; d < HD; ++d) s = fmaf((float)q[d], (float)k[j * k_row + d], s);
      s = j < j1 ? s * scale2 : -INFINITY;
      float most = s;
      for (int x = 32; x > 0; x >>= 1) most = fmaxf(most, __shfl_xor(most, x, 64));
      const float mn = fmaxf(m, most), ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = exp2f(m - ref), p = j < j1 ? exp2f(s - ref) : 0.f;
      float sum = p;
      for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x, 64);
      l = l * alpha + sum;
      m = mn;
      for (int i = 0; i < HD / 64; ++i) o[i] *= alpha;
      for (int t = 0; t < min(64, j1 - jb); ++t) {
        const float pt = __shfl(p, t, 64);
        for (int i = 0; i < HD / 64; ++i) o[i] = fmaf(pt, (float)v[(jb + t) * v_row + lane + 64 * i], o[i]);
      }
    }
  }
};

// One wave a (query, head) row.
template <typename T, int HD>
__global__ __launch_bounds__(256) void window_row_kernel(WindowArgs a) {
  constexpr int R = 4;
  const nemo_attention_batch& b = a.b;
  const int i = tile_request(b, a.group, R, blockIdx.x);
  if (i < 0) return;
  const Request r(b, i);
  const int row = (blockIdx.x - tile_base(b, a.group, R, i)) * R + (threadIdx.x >> 6);
  if (row >= r.queries * a.group) return;
  const int qi = row / a.group, h = blockIdx.y * a.group + row % a.group, lane = threadIdx.x & 63;
  const T* q = (const T*)b.q + (int64_t)(r.q0 + qi) * b.q_row + h * b.q_head;
  const T* k = (const T*)b.k + r.kv0 * b.k_row + blockIdx.y * b.k_head;
  const T* v = (const T*)b.v + r.kv0 * b.v_row + blockIdx.y * b.v_head;
  T* out = (T*)b.out + (int64_t)(r.q0 + qi) * b.out_row + h * b.out_head;
  const Seen seen(a, r.keys - r.queries + qi, r.keys);
  OneRow<T, HD> acc;
  acc.keys(q, k, b.k_row, v, b.v_row, 0, seen.sinks, a.scale2);
  acc.keys(q, k, b.k_row, v, b.v_row, seen.lo, seen.hi, a.scale2);
  for (int c = 0; c < HD / 64; ++c) out[lane + 64 * c] = (T)(acc.l == 0.f ? 0.f : acc.o[c] / acc.l);
}

}  // namespace

int window_splits(const nemo_attention_config& c, int count, int64_t q_rows, int64_t max_kv) { return 1; }

size_t window_workspace(const nemo_attention_config& c, int count, int64_t q_rows, int64_t max_kv) { return 0; }

hipError_t launch_window_attention(const nemo_attention_config& c, const nemo_attention_batch& b, hipStream_t stream) {
  if (b.count == 0 || b.q_rows == 0) return hipSuccess;
  WindowArgs a{b, c.q_heads / c.kv_heads, 0, 0, 0, 0.f};
  auto bound = [](int v) { return v < 0 ? kUnbounded : std::min(v, kUnbounded); };
  a.left = bound(c.left);
  a.right = bound(c.right);
  a.sinks = std::min(c.sinks, kUnbounded);
  a.scale2 = (c.scale > 0.f ? c.scale : 1.0f / sqrtf((float)c.head_dim)) * 1.4426950408889634f;
  const dim3 grid((unsigned)(b.q_rows * a.group / 4 + b.count), c.kv_heads);
  if (c.type == NEMO_TYPE_F16) {
    if (c.head_dim == 64) window_row_kernel<half_t, 64><<<grid, 256, 0, stream>>>(a);
    else window_row_kernel<half_t, 128><<<grid, 256, 0, stream>>>(a);
  } else {
    if (c.head_dim == 64) window_row_kernel<bf16_t, 64><<<grid, 256, 0, stream>>>(a);
    else window_row_kernel<bf16_t, 128><<<grid, 256, 0, stream>>>(a);
  }
  return hipGetLastError();
}

}  // namespace nemo
