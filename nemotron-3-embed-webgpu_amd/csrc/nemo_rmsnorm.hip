// Residual addition, RMSNorm and 8-bit output with scales for gfx950: h = x +
// delta, y = h / sqrt(mean(h^2) + eps) * w, y8 = round(y / s) with s = max |y|
// / 127 (bytes) or / 448 (8-bit floats) over a row or a group of columns.
//
// The row's factor cancels in y / s = h w top / max |h w|, whose seven roundings
// in 32 bits (h and its product with w, here and in the maximum, the quotient,
// and two products with that) leave it within 7 2^-24 of itself. Next to a
// border between two codes that decides wrongly a few times in a million
// values, so each is coded from both ends of 2^-21 around it, and a wave in
// which two codes differ (about one in a hundred) takes its values again in 64
// bits, with what the sum x + delta of 32-bit values lost, and rounds once. (The
// sum of 16-bit values is exact but for a delta some 2^-13 of its x and
// smaller.) In 64 bits throughout, 16384 x 8192 bf16 to 8-bit floats with scales
// of 128 columns took 226 us.
//
// Bound by memory: each value is read and written once, 16 bytes a lane. Those
// 16384 rows, 944 MB, take 177 us call after call (5.3 TB/s; a copy reaches 4.9
// to 5.4), 182 at the least and 195 mostly where a trace sets the calls apart;
// 2399 x 2048 f16 to bytes and f16 11.6 and 12.7 there, 44 MB that 5.4 TB/s
// would take in 8.2.
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
__device__ __forceinline__ uint64_t magnitude(double v) {
  return __builtin_bit_cast(uint64_t, v) & 0x7fffffffffffffffull;
}
__device__ __forceinline__ uint32_t lanes_max(uint32_t v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
  return v;
}
__device__ __forceinline__ uint64_t lanes_max(uint64_t v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v = max(v, (uint64_t)__shfl_xor((unsigned long long)v, o, 64));
  return v;
}

// Codes of four quotients: bytes, or 8-bit floats (448 (1 + 2^-21) rounds to 448).
__device__ __forceinline__ uint32_t code4(bool bytes, float a, float b, float c, float d) {
  if (bytes)
    return ((uint32_t)(int)rintf(a) & 255u) | ((uint32_t)(int)rintf(b) & 255u) << 8 |
           ((uint32_t)(int)rintf(c) & 255u) << 16 | (uint32_t)(int)rintf(d) << 24;
  const int low = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, low, true);
}

__device__ __forceinline__ uint8_t code1(bool bytes, float v) {
  if (bytes) return (uint8_t)(int)rintf(v);
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false);
}

// v with its last bit set where 32 bits do not hold it, rounded to zero before:
// a code of that is v's own.
__device__ __forceinline__ float odd(double v) {
  const float f = (float)v;
  uint32_t bits = __float_as_uint(f);
  if ((double)f != v) bits = (bits - (fabs((double)f) > fabs(v) ? 1 : 0)) | 1;
  return __uint_as_float(bits);
}

// The scale of values h w `factor` whose largest |h w| is `peak` (its bits), and
// factors that take h w to below and above its quotient with it.
struct Quantizer {
  float scale, low, high;
  bool unsure;  // h w may be below the range where 32 bits hold its quotient
  __device__ __forceinline__ Quantizer(uint32_t peak, float factor, float top) {
    const float p = __uint_as_float(peak);
    scale = p * factor / top;
    const float inv = scale == 0.f ? 0.f : top / p;
    low = inv * (1 - 0x1p-21f);
    high = inv * (1 + 0x1p-21f);
    unsure = p < 0x1p-100f;
  }
};
// The same in 64 bits.
struct Quantizer64 {
  float scale;
  double inv;
  __device__ __forceinline__ Quantizer64(uint64_t peak, float factor, double top) {
    const double p = __builtin_bit_cast(double, peak);
    scale = (float)(p * factor / top);
    inv = scale == 0.f ? 0.0 : top / p;
  }
};

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
  __shared__ float part[16];
  __shared__ uint32_t peaks[16];
  __shared__ uint64_t peaks64[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = WAVES >= 4 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (4 / WAVES) + wave / WAVES;
  if (row >= a.rows) return;  // rows of one wave only: no barrier is left behind
  const int first = 8 * (64 * (wave % WAVES) + lane);
  const T* x = (const T*)a.x + row * a.x_row;
  const T* delta = (const T*)a.delta + row * a.delta_row;
  constexpr bool LOST = sizeof(T) == 4;
  float h[NV][8], lost[LOST ? NV : 1][8] = {};  // h and what its rounding left out
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
        for (int e = 0; e < 8; ++e) {
          const float from = h[i][e], add = (float)v[e];
          h[i][e] = from + add;
          if constexpr (LOST) {
            const float added = h[i][e] - from;
            lost[i][e] = (from - (h[i][e] - added)) + (add - added);
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(h[i][e], h[i][e], sum);
  auto exact = [&](int i, int e) { return LOST ? (double)h[i][e] + (double)lost[LOST ? i : 0][e] : (double)h[i][e]; };
  sum = wave_sum(sum);
  if constexpr (WAVES > 1) {
    if (lane == 0) part[wave] = sum;
    __syncthreads();
    sum = part[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum += part[w];
  }
  const float inv = 1.0f / sqrtf(sum / (float)a.hidden + a.epsilon);
  float w[NV][8];
  uint32_t peak[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = first + 512 * WAVES * i;
    peak[i] = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[i][e] = 1.f;
    if (c >= a.hidden) continue;
    if (a.sum) {
      vec v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (T)h[i][e];
      *(vec*)((T*)a.sum + row * a.sum_row + c) = v;
    }
    if (a.weight) {
      const float4v w0 = *(const float4v*)(a.weight + c), w1 = *(const float4v*)(a.weight + c + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[i][e] = w0[e], w[i][4 + e] = w1[e];
    }
    if (a.y) {
      vec v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (T)(h[i][e] * inv * w[i][e]);
      *(vec*)((T*)a.y + row * a.y_row + c) = v;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) peak[i] = max(peak[i], magnitude(h[i][e] * w[i][e]));
  }
  if (!a.y8) return;
  // A row's largest value, of which each wave also leaves the exact product; a
  // group's. Products that 32 bits order otherwise than they are lie at most 4
  // units in the last place below the largest: the lanes that have one take
  // its exact product, mostly a single lane. (Without the test of each value
  // the compiler holds all exact products from here on: 16384 x 8192 bf16 176
  // -> 192 us.)
  if (a.group == 0) {
    uint32_t own = peak[0];
#pragma unroll
    for (int i = 1; i < NV; ++i) own = max(own, peak[i]);
    uint32_t most = lanes_max(own, 64);
    if constexpr (WAVES > 1) {
      constexpr uint32_t NEAR = 8;  // (h and its product with w round, for both, by 2^-24 at most)
      const uint64_t near = __builtin_amdgcn_ballot_w64(own + NEAR >= most);
      uint64_t most64 = 0;
      if (own + NEAR >= most) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (magnitude(h[i][e] * w[i][e]) + NEAR >= most)
              most64 = max(most64, magnitude(exact(i, e) * (double)w[i][e]));
      }
      if (near & (near - 1)) most64 = lanes_max(most64, 64);
      if (lane == __builtin_ctzll(near)) {
        peaks[wave] = most;
        peaks64[wave] = most64;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < WAVES; ++k) most = max(most, peaks[k]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) peak[i] = most;
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) peak[i] = lanes_max(peak[i], a.group / 8);
  }
  const bool bytes = a.type8 == NEMO_TYPE_I8;
  const float top = bytes ? 127.f : 448.f;
  float* scales = a.scales + row * a.scales_row;
  auto put = [&](int c, float scale, u32x2 codes) {
    if (a.group ? c % a.group == 0 : c == 0) scales[a.group ? c / a.group : 0] = scale;
    *(u32x2*)((uint8_t*)a.y8 + row * a.y8_row + c) = codes;
  };
  bool unsure = false;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = first + 512 * WAVES * i;
    if (c >= a.hidden) continue;
    const Quantizer q(peak[i], inv, top);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = h[i][e] * w[i][e];
    u32x2 codes;
    unsure |= q.unsure;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float* u = v + 4 * j;
      codes[j] = code4(bytes, u[0] * q.low, u[1] * q.low, u[2] * q.low, u[3] * q.low);
      unsure |= codes[j] != code4(bytes, u[0] * q.high, u[1] * q.high, u[2] * q.high, u[3] * q.high);
    }
    put(c, q.scale, codes);
  }
  if (!__builtin_amdgcn_ballot_w64(unsure)) return;
  uint64_t peak64[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    peak64[i] = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) peak64[i] = max(peak64[i], magnitude(exact(i, e) * (double)w[i][e]));
  }
  if (a.group) {
#pragma unroll
    for (int i = 0; i < NV; ++i) peak64[i] = lanes_max(peak64[i], a.group / 8);
  } else {
    uint64_t most = 0;
    if constexpr (WAVES > 1) {
#pragma unroll
      for (int k = 0; k < WAVES; ++k) most = max(most, peaks64[k]);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) most = max(most, peak64[i]);
      most = lanes_max(most, 64);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) peak64[i] = most;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = first + 512 * WAVES * i;
    if (c >= a.hidden) continue;
    const Quantizer64 q(peak64[i], inv, top);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = odd(exact(i, e) * (double)w[i][e] * q.inv);
    put(c, q.scale, u32x2{code4(bytes, v[0], v[1], v[2], v[3]), code4(bytes, v[4], v[5], v[6], v[7])});
  }
}

// Any alignment and stride: a lane holds 8 values of a row of up to 512, one
// wave a row, value i of column 64 i + lane. All in 64 bits (4096 x 147 f32 to
// 8-bit floats 6.9 us, by the kernel below 10).
template <typename T>
__global__ __launch_bounds__(256) void norm8_values_kernel(nemo_norm_args a) {
  constexpr int NV = 8;
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  const T* x = (const T*)a.x + row * a.x_row;
  const T* delta = (const T*)a.delta + row * a.delta_row;
  double h[NV];
  float w[NV], sum = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = 64 * i + lane;
    h[i] = c < a.hidden ? (double)(float)x[c] + (a.delta ? (double)(float)delta[c] : 0.0) : 0.0;
    w[i] = a.weight && c < a.hidden ? a.weight[c] : 1.f;
    sum = fmaf((float)h[i], (float)h[i], sum);
  }
  sum = wave_sum(sum);
  const float inv = 1.0f / sqrtf(sum / (float)a.hidden + a.epsilon);
  uint64_t peak[NV], most = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = 64 * i + lane;
    peak[i] = magnitude(h[i] * (double)w[i]);
    most = max(most, peak[i]);
    if (c >= a.hidden) continue;
    if (a.sum) ((T*)a.sum)[row * a.sum_row + c] = (T)(float)h[i];
    if (a.y) ((T*)a.y)[row * a.y_row + c] = (T)((float)h[i] * inv * w[i]);
  }
  if (!a.y8) return;
  most = lanes_max(most, 64);
  const bool bytes = a.type8 == NEMO_TYPE_I8;
#pragma unroll
  for (int i = 0; i < NV; i += 2) {
    if (a.group == 128) peak[i] = peak[i + 1] = max(peak[i], peak[i + 1]);
#pragma unroll
    for (int k = i; k < i + 2; ++k) {
      const int c = 64 * k + lane;
      const uint64_t top = a.group ? lanes_max(peak[k], min(a.group, 64)) : most;
      if (c >= a.hidden) continue;
      const Quantizer64 q(top, inv, bytes ? 127.0 : 448.0);
      if (a.group ? c % a.group == 0 : c == 0) a.scales[row * a.scales_row + (a.group ? c / a.group : 0)] = q.scale;
      ((uint8_t*)a.y8)[row * a.y8_row + c] = code1(bytes, odd(h[k] * (double)w[k] * q.inv));
    }
  }
}

// Longer rows of any alignment and stride: a workgroup reads its row once for
// the norm, once more for a whole row's scale, and once to write (a lane what it
// has just read). Codes are decided as above. Bound by its loads and stores of
// single values, some ten each (4096 x 3145 f32 to 8-bit floats 67 us, 2.5 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void norm8_any_kernel(nemo_norm_args a) {
  __shared__ float part[4];
  __shared__ uint64_t peaks[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.x_row;
  const T* delta = a.delta ? (const T*)a.delta + row * a.delta_row : nullptr;
  float sum = 0.f;
  for (int c = threadIdx.x; c < a.hidden; c += 256) {
    const float v = (float)x[c] + (delta ? (float)delta[c] : 0.f);
    sum = fmaf(v, v, sum);
  }
  sum = wave_sum(sum);
  if (lane == 0) part[wave] = sum;
  __syncthreads();
  sum = part[0] + part[1] + part[2] + part[3];
  const float inv = 1.0f / sqrtf(sum / (float)a.hidden + a.epsilon);
  auto exact = [](float from, float add, float w) { return ((double)from + (double)add) * (double)w; };
  uint64_t most = 0;
  if (a.y8 && a.group == 0) {
    float near = -1.f;  // the largest magnitude so far less what 32 bits may be off by
    for (int c = threadIdx.x; c < a.hidden; c += 256) {
      const float from = (float)x[c], add = delta ? (float)delta[c] : 0.f, w = a.weight ? a.weight[c] : 1.f;
      const float v = fabsf((from + add) * w);
      if (v < near) continue;
      near = fmaxf(near, v * (1 - 0x1p-20f) - 0x1p-140f);
      most = max(most, magnitude(exact(from, add, w)));
    }
    most = lanes_max(most, 64);
    if (lane == 0) peaks[wave] = most;
    __syncthreads();
    for (int w = 0; w < 4; ++w) most = max(most, peaks[w]);
  }
  const bool bytes = a.type8 == NEMO_TYPE_I8;
  const float top = bytes ? 127.f : 448.f;
  float* scales = a.y8 ? a.scales + row * a.scales_row : nullptr;
  uint8_t* y8 = (uint8_t*)a.y8 + row * a.y8_row;
  const int width = a.group ? a.group : 128;  // columns of a wave's step, up to 2 a lane
  for (int at = width * wave; at < a.hidden; at += 4 * width) {
    float from[2], add[2], h[2], w[2];
    uint32_t peak = 0;
    bool in[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = at + lane + 64 * i;
      in[i] = lane + 64 * i < width && c < a.hidden;
      from[i] = in[i] ? (float)x[c] : 0.f;
      add[i] = in[i] && delta ? (float)delta[c] : 0.f;
      w[i] = in[i] && a.weight ? a.weight[c] : 1.f;
      h[i] = from[i] + add[i];
      peak = max(peak, magnitude(h[i] * w[i]));
      if (in[i] && a.sum) ((T*)a.sum)[row * a.sum_row + c] = (T)h[i];
      if (in[i] && a.y) ((T*)a.y)[row * a.y_row + c] = (T)(h[i] * inv * w[i]);
    }
    if (!a.y8) continue;
    const double most_value = __builtin_bit_cast(double, most);
    const Quantizer q(a.group ? lanes_max(peak, 64) : magnitude((float)most_value), inv, top);
    uint8_t code[2];
    float scale = q.scale;
    bool unsure = q.unsure;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      code[i] = code1(bytes, h[i] * w[i] * q.low);
      unsure |= code[i] != code1(bytes, h[i] * w[i] * q.high);
    }
    if (__builtin_amdgcn_ballot_w64(unsure)) {
      const uint64_t own = max(magnitude(exact(from[0], add[0], w[0])), magnitude(exact(from[1], add[1], w[1])));
      const Quantizer64 q64(a.group ? lanes_max(own, 64) : most, inv, top);
      scale = q64.scale;
#pragma unroll
      for (int i = 0; i < 2; ++i) code[i] = code1(bytes, odd(exact(from[i], add[i], w[i]) * q64.inv));
    }
    if (lane == 0 && (a.group || at == 0)) scales[a.group ? at / a.group : 0] = scale;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (in[i]) y8[at + lane + 64 * i] = code[i];
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
  if (!vectors && a.hidden <= 512)
    norm8_values_kernel<T><<<(rows + 3) / 4, 256, 0, stream>>>(a);
  else if (!vectors)
    norm8_any_kernel<T><<<rows, 256, 0, stream>>>(a);
  else if (blocks <= 64)
    norm8_kernel<T, 1, 1><<<(rows + 3) / 4, 256, 0, stream>>>(a);
  else if (blocks <= 256)
    norm8_kernel<T, 4, 1><<<rows, 256, 0, stream>>>(a);
  else if (blocks <= 512)
    norm8_kernel<T, 4, 2><<<rows, 256, 0, stream>>>(a);
  else if (blocks <= 1024 && sizeof(T) == 2)  // (16384 x 8192: 4 waves of 4 blocks 219 us, 8 of 2 177, 16 of one 188)
    norm8_kernel<T, 8, 2><<<rows, 512, 0, stream>>>(a);
  else if (blocks <= 1024)  // (what its sums lost takes registers too: 4096 x 8192, 8 of 2 88 us, 16 of one 81)
    norm8_kernel<T, 16, 1><<<rows, 1024, 0, stream>>>(a);
  else if (blocks <= 2048)  // (4096 x 16384, 16 waves: f32, 4 blocks 256 us, 2 180; bf16 140, 98)
    norm8_kernel<T, 16, 2><<<rows, 1024, 0, stream>>>(a);
  else
    norm8_kernel<T, 16, 4><<<rows, 1024, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_norm8(const nemo_norm_args& args, hipStream_t stream) {
  // Rows of a launch: with up to 1024 threads a row, fewer threads than the 2^32 that a grid may not reach.
  constexpr int64_t kLaunchRows = 1 << 21;
  const int64_t size = args.type == NEMO_TYPE_F32 ? 4 : 2;
  for (int64_t row = 0; row < args.rows; row += kLaunchRows) {
    nemo_norm_args a = args;
    auto skip = [row](auto* p, int64_t bytes) { return p ? (decltype(p))((uintptr_t)p + row * bytes) : p; };
    a.rows = std::min(kLaunchRows, args.rows - row);
    a.x = skip(a.x, a.x_row * size);
    a.delta = skip(a.delta, a.delta_row * size);
    a.sum = skip(a.sum, a.sum_row * size);
    a.y = skip(a.y, a.y_row * size);
    a.y8 = skip(a.y8, a.y8_row);
    a.scales = skip(a.scales, a.scales_row * 4);
    hipError_t e = hipErrorInvalidValue;
    switch (a.type) {
      case NEMO_TYPE_F32: e = launch_norm_type<float>(a, stream); break;
      case NEMO_TYPE_F16: e = launch_norm_type<half_t>(a, stream); break;
      case NEMO_TYPE_BF16: e = launch_norm_type<bf16_t>(a, stream); break;
    }
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace nemo
