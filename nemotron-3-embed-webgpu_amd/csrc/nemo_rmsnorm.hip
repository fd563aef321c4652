// Residual addition, RMSNorm and 8-bit output with scales for gfx950: h = x +
// delta, y = h / sqrt(mean(h^2) + eps) * w, y8 = round(y / s) with s = max |y|
// / 127 (bytes) or / 448 (8-bit floats) over a row or a group of columns.
#include <algorithm>

#include "nemo_operators.h"

namespace nemo {

namespace {

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// The largest magnitude, as its bits: they order as the magnitudes do, with
// NaN above infinity, so a NaN is not lost as a floating maximum would.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t lanes_max(uint32_t v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
  return v;
}

// The scale of values up to the magnitude `peak`, and y / scale = y * pre *
// inv. Peaks below 2^-100 are raised by 2^64 first: 127 / peak would overflow.
struct Quantizer {
  float scale, pre, inv;
  __device__ __forceinline__ Quantizer(uint32_t bits, float top) {
    const float peak = __uint_as_float(bits);
    pre = peak < 0x1p-100f ? 0x1p64f : 1.0f;
    scale = peak / top;
    inv = bits == 0 ? 0.f : top / (peak * pre);
  }
  __device__ __forceinline__ float operator()(float y) const { return y * pre * inv; }
};

__device__ __forceinline__ uint32_t to_i8(float v) { return (uint32_t)(int)rintf(v) & 255u; }
// E4M3 codes of two values; a quotient can round past 448, to which it is cut.
__device__ __forceinline__ uint32_t to_e4m3(float a, float b) {
  a = a == a ? __builtin_amdgcn_fmed3f(a, -448.f, 448.f) : a;
  b = b == b ? __builtin_amdgcn_fmed3f(b, -448.f, 448.f) : b;
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}

template <typename T>
struct Vec8 {
  typedef T type __attribute__((ext_vector_type(8)));
};

// Rows of up to 512 WAVES NV values, 16-byte vectors: WAVES waves of a
// workgroup hold a row in registers, lane l of wave w the NV blocks of 8
// columns from 8 (64 (WAVES i + w) + l). A lane writes only columns that it
// read before, so sum and y may replace x and delta.
template <typename T, int WAVES, int NV>
__global__ __launch_bounds__(WAVES > 4 ? 64 * WAVES : 256) void norm8_kernel(nemo_norm_args a) {
  typedef typename Vec8<T>::type vec;
  __shared__ float part[2][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = WAVES >= 4 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (4 / WAVES) + wave / WAVES;
  if (row >= a.rows) return;  // rows of one wave only: no barrier is left behind
  const int first = 8 * (64 * (wave % WAVES) + lane);
  const T* x = (const T*)a.x + row * a.x_row;
  const T* delta = (const T*)a.delta + row * a.delta_row;
  float h[NV][8];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = first + 512 * WAVES * i;
    if (c < a.hidden) {
      const vec v = *(const vec*)(x + c);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] = (float)v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] = 0.f;
    }
  }
  if (a.delta) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = first + 512 * WAVES * i;
      if (c < a.hidden) {
        const vec v = *(const vec*)(delta + c);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] += (float)v[e];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(h[i][e], h[i][e], sum);
  sum = wave_sum(sum);
  if constexpr (WAVES > 1) {
    if (lane == 0) part[0][wave] = sum;
    __syncthreads();
    sum = part[0][0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum += part[0][w];
  }
  const float inv = 1.0f / sqrtf(sum / (float)a.hidden + a.epsilon);
  uint32_t peak[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = first + 512 * WAVES * i;
    peak[i] = 0;
    if (c >= a.hidden) continue;
    if (a.sum) {
      vec v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (T)h[i][e];
      *(vec*)((T*)a.sum + row * a.sum_row + c) = v;
    }
    float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
    if (a.weight) {
      const float4v w0 = *(const float4v*)(a.weight + c), w1 = *(const float4v*)(a.weight + c + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = w0[e], w[4 + e] = w1[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[i][e] = h[i][e] * inv * w[e];
      peak[i] = max(peak[i], magnitude(h[i][e]));
    }
    if (a.y) {
      vec v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (T)h[i][e];
      *(vec*)((T*)a.y + row * a.y_row + c) = v;
    }
  }
  if (!a.y8) return;
  if (a.group == 0) {
    uint32_t most = peak[0];
#pragma unroll
    for (int i = 1; i < NV; ++i) most = max(most, peak[i]);
    most = lanes_max(most, 64);
    if constexpr (WAVES > 1) {
      if (lane == 0) part[1][wave] = __uint_as_float(most);
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) most = max(most, __float_as_uint(part[1][w]));
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) peak[i] = most;
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) peak[i] = lanes_max(peak[i], a.group / 8);
  }
  const float top = a.type8 == NEMO_TYPE_I8 ? 127.f : 448.f;
  float* scales = a.scales + row * a.scales_row;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = first + 512 * WAVES * i;
    if (c >= a.hidden) continue;
    const Quantizer q(peak[i], top);
    if (a.group ? c % a.group == 0 : c == 0) scales[a.group ? c / a.group : 0] = q.scale;
    u32x2 o;
    if (a.type8 == NEMO_TYPE_I8) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        o[j] = to_i8(q(h[i][4 * j])) | to_i8(q(h[i][4 * j + 1])) << 8 | to_i8(q(h[i][4 * j + 2])) << 16 |
               to_i8(q(h[i][4 * j + 3])) << 24;
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        o[j] = to_e4m3(q(h[i][4 * j]), q(h[i][4 * j + 1])) | to_e4m3(q(h[i][4 * j + 2]), q(h[i][4 * j + 3])) << 16;
    }
    *(u32x2*)((uint8_t*)a.y8 + row * a.y8_row + c) = o;
  }
}

// Any sizes, strides and alignments: a workgroup reads its row once for the
// norm, once more for a whole row's scale, and once to write (a lane what it
// has just read).
template <typename T>
__global__ __launch_bounds__(256) void norm8_any_kernel(nemo_norm_args a) {
  __shared__ float part[2][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.x_row;
  const T* delta = a.delta ? (const T*)a.delta + row * a.delta_row : nullptr;
  auto load = [&](int c) { return (float)x[c] + (delta ? (float)delta[c] : 0.f); };
  float sum = 0.f;
  for (int c = threadIdx.x; c < a.hidden; c += 256) {
    const float v = load(c);
    sum = fmaf(v, v, sum);
  }
  sum = wave_sum(sum);
  if (lane == 0) part[0][wave] = sum;
  __syncthreads();
  sum = part[0][0] + part[0][1] + part[0][2] + part[0][3];
  const float inv = 1.0f / sqrtf(sum / (float)a.hidden + a.epsilon);
  auto normed = [&](float v, int c) { return v * inv * (a.weight ? a.weight[c] : 1.f); };
  uint32_t most = 0;
  if (a.y8 && a.group == 0) {
    for (int c = threadIdx.x; c < a.hidden; c += 256) most = max(most, magnitude(normed(load(c), c)));
    most = lanes_max(most, 64);
    if (lane == 0) part[1][wave] = __uint_as_float(most);
    __syncthreads();
    for (int w = 0; w < 4; ++w) most = max(most, __float_as_uint(part[1][w]));
  }
  const float top = a.type8 == NEMO_TYPE_I8 ? 127.f : 448.f;
  float* scales = a.y8 ? a.scales + row * a.scales_row : nullptr;
  const int width = a.group ? a.group : 128;  // columns of a wave's step, up to 2 a lane
  for (int at = width * wave; at < a.hidden; at += 4 * width) {
    float h[2], y[2];
    uint32_t peak = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = at + lane + 64 * i;
      const bool in = lane + 64 * i < width && c < a.hidden;
      h[i] = in ? load(c) : 0.f;
      y[i] = in ? normed(h[i], c) : 0.f;
      peak = max(peak, magnitude(y[i]));
    }
    peak = a.group ? lanes_max(peak, 64) : most;
    const Quantizer q(peak, top);
    if (a.y8 && lane == 0 && (a.group || at == 0)) scales[a.group ? at / a.group : 0] = q.scale;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = at + lane + 64 * i;
      if (lane + 64 * i >= width || c >= a.hidden) continue;
      if (a.sum) ((T*)a.sum)[row * a.sum_row + c] = (T)h[i];
      if (a.y) ((T*)a.y)[row * a.y_row + c] = (T)y[i];
      if (a.y8) {
        const float v = q(y[i]);
        ((uint8_t*)a.y8)[row * a.y8_row + c] = (uint8_t)(a.type8 == NEMO_TYPE_I8 ? to_i8(v) : to_e4m3(v, 0.f));
      }
    }
  }
}

template <typename T>
hipError_t launch_norm_type(const nemo_norm_args& a, hipStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const int blocks = (a.hidden + 7) / 8;  // of 8 columns
  auto fits = [](const void* p, int64_t row) { return !p || (((uintptr_t)p & 15) == 0 && row % V == 0); };
  const bool vectors = a.hidden % 8 == 0 && fits(a.x, a.x_row) && fits(a.delta, a.delta_row) &&
                       fits(a.sum, a.sum_row) && fits(a.y, a.y_row) && ((uintptr_t)a.weight & 15) == 0 &&
                       (!a.y8 || (((uintptr_t)a.y8 & 7) == 0 && a.y8_row % 8 == 0)) && blocks <= 64 * 16 * 4;
  const unsigned rows = (unsigned)a.rows;
  if (!vectors)
    norm8_any_kernel<T><<<rows, 256, 0, stream>>>(a);
  else if (blocks <= 64)
    norm8_kernel<T, 1, 1><<<(rows + 3) / 4, 256, 0, stream>>>(a);
  else if (blocks <= 256)
    norm8_kernel<T, 4, 1><<<rows, 256, 0, stream>>>(a);
  else if (blocks <= 512)
    norm8_kernel<T, 4, 2><<<rows, 256, 0, stream>>>(a);
  else if (blocks <= 1024)
    norm8_kernel<T, 4, 4><<<rows, 256, 0, stream>>>(a);
  else
    norm8_kernel<T, 16, 4><<<rows, 1024, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_norm8(const nemo_norm_args& args, hipStream_t stream) {
  if (args.rows == 0) return hipSuccess;
  switch (args.type) {
    case NEMO_TYPE_F32: return launch_norm_type<float>(args, stream);
    case NEMO_TYPE_F16: return launch_norm_type<half_t>(args, stream);
    case NEMO_TYPE_BF16: return launch_norm_type<bf16_t>(args, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace nemo
