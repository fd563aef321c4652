// Rotary positions on heads of any layout for gfx950: (a, b) -> m (a cos - b
// sin, a sin + b cos) with the angle position * f_i, whose whole turns are
// taken off in 64 bits (a position of 2^20 leaves an angle in 32 bits some
// 0.06 rad off), so the sine and cosine are of an angle within half a turn.
//
// Bound by memory, each head read and written once, once a thread's angles
// serve several heads: 32768 tokens of 40 bf16 heads of 128 at positions up to
// 2^20, 671 MB, take 118 us (5.7 TB/s; a copy reaches 4.9 to 5.4), 5001 tokens
// of 15 f32 heads of 96 12.8 (medians 121 and 13.7), one token 2.3.
#include <algorithm>

#include "nemo_operators.h"

namespace nemo {

namespace {

struct RopeArgs {
  nemo_rope_heads q, k;  // k.heads 0: none
  const double* turns;
  const int64_t* positions;
  int64_t base, rows;
  float magnitude;
  int head_dim, pairs, rest;  // rest: values behind the pairs that are copied, none where heads are turned in place
  bool half;
};

// Cosine and sine, scaled, of pair i at position p.
__device__ __forceinline__ float2 rope_angle(const RopeArgs& a, int i, double p) {
  double t = p * a.turns[i];
  t -= rint(t);
  float s, c;
  sincospif(2.0f * (float)t, &s, &c);
  return make_float2(c * a.magnitude, s * a.magnitude);
}

template <typename T>
__device__ __forceinline__ void rope_head(const RopeArgs& a, int64_t t, int h, const T*& x, T*& y) {
  const bool key = h >= a.q.heads;
  const nemo_rope_heads& s = key ? a.k : a.q;
  const int64_t i = key ? h - a.q.heads : h;
  x = (const T*)s.x + t * s.x_row + i * s.x_head;
  y = (T*)s.y + t * s.y_row + i * s.y_head;
}

__device__ __forceinline__ double rope_position(const RopeArgs& a, int64_t t) {
  return (double)(a.base + (a.positions ? a.positions[t] : t));
}

// Any sizes, strides and alignments: a thread turns one pair or copies one
// value of one head.
template <typename T>
__global__ __launch_bounds__(256) void rope_any_kernel(RopeArgs a) {
  const int units = a.pairs + a.rest;
  const int64_t heads = a.q.heads + a.k.heads, total = a.rows * heads * units;
  for (int64_t n = blockIdx.x * 256ll + threadIdx.x; n < total; n += gridDim.x * 256ll) {
    const int u = (int)(n % units);
    const int64_t th = n / units, t = th / heads;
    const T* x;
    T* y;
    rope_head(a, t, (int)(th - t * heads), x, y);
    if (u >= a.pairs) {
      y[a.pairs + u] = x[a.pairs + u];
      continue;
    }
    const float2 cs = rope_angle(a, u, rope_position(a, t));
    const int i = a.half ? u : 2 * u, j = a.half ? u + a.pairs : 2 * u + 1;
    const float e = (float)x[i], o = (float)x[j];
    y[i] = (T)(e * cs.x - o * cs.y);
    y[j] = (T)(e * cs.y + o * cs.x);
  }
}

// Vectors of E values, up to 16 bytes. A head is `units` units: interleaved, one
// vector each; half, first the vectors of the pairs' first values, each with
// that of their second ones, then the vectors that are copied. A thread
// computes the angles of its unit once and turns it in every `slots`-th head
// of its token.
template <typename T, int E>
__global__ __launch_bounds__(256) void rope_vector_kernel(RopeArgs a, int units, int slots, int tokens) {
  typedef T vec __attribute__((ext_vector_type(E)));
  const int per = units * slots, u = threadIdx.x % units;
  const int64_t t = (int64_t)blockIdx.x * tokens + threadIdx.x / per;
  if ((int)threadIdx.x >= tokens * per || t >= a.rows) return;
  const int slot = threadIdx.x % per / units, heads = a.q.heads + a.k.heads;
  const int turned = a.half ? a.pairs / E : 2 * a.pairs / E;  // units that hold pairs
  if (u >= turned) {
    const int d = a.half ? a.pairs + E * u : E * u;
    for (int h = slot; h < heads; h += slots) {
      const T* x;
      T* y;
      rope_head(a, t, h, x, y);
      *(vec*)(y + d) = *(const vec*)(x + d);
    }
    return;
  }
  const double p = rope_position(a, t);
  if (a.half) {
    float2 cs[E];
#pragma unroll
    for (int e = 0; e < E; ++e) cs[e] = rope_angle(a, E * u + e, p);
    for (int h = slot; h < heads; h += slots) {
      const T* x;
      T* y;
      rope_head(a, t, h, x, y);
      const vec v = *(const vec*)(x + E * u), w = *(const vec*)(x + a.pairs + E * u);
      vec r, s;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        r[e] = (T)((float)v[e] * cs[e].x - (float)w[e] * cs[e].y);
        s[e] = (T)((float)v[e] * cs[e].y + (float)w[e] * cs[e].x);
      }
      *(vec*)(y + E * u) = r;
      *(vec*)(y + a.pairs + E * u) = s;
    }
    return;
  }
  if constexpr (E > 1) {
    float2 cs[E / 2];
#pragma unroll
    for (int e = 0; e < E / 2; ++e) cs[e] = rope_angle(a, E / 2 * u + e, p);
    for (int h = slot; h < heads; h += slots) {
      const T* x;
      T* y;
      rope_head(a, t, h, x, y);
      const vec v = *(const vec*)(x + E * u);
      vec r;
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        r[2 * e] = (T)((float)v[2 * e] * cs[e].x - (float)v[2 * e + 1] * cs[e].y);
        r[2 * e + 1] = (T)((float)v[2 * e] * cs[e].y + (float)v[2 * e + 1] * cs[e].x);
      }
      *(vec*)(y + E * u) = r;
    }
  }
}

bool aligned_heads(const nemo_rope_heads& s, int E, int bytes) {
  return (((uintptr_t)s.x | (uintptr_t)s.y) & (bytes - 1)) == 0 &&
         s.x_row % E == 0 && s.x_head % E == 0 && s.y_row % E == 0 && s.y_head % E == 0;
}

// By vectors of E values, or narrower ones that the sizes, strides and
// addresses allow (8192 tokens of 32 bf16 heads of 128, 40 of them turned by
// halves, vectors of 4: 49 us, single values by rope_any_kernel 122; 102 turned,
// vectors of 1 80 : 103).
template <typename T, int E = 16 / sizeof(T)>
hipError_t launch_rope_type(const RopeArgs& a, hipStream_t stream) {
  const int heads = a.q.heads + a.k.heads, rotary = 2 * a.pairs, bytes = E * sizeof(T);
  const bool vectors = a.head_dim % E == 0 && rotary % E == 0 && (a.half ? a.pairs % E == 0 : E > 1) &&
                       aligned_heads(a.q, E, bytes) && (!a.k.heads || aligned_heads(a.k, E, bytes));
  const int units = (a.half ? a.pairs : rotary) / E + a.rest / E;
  if (vectors && units <= 256) {
    const int slots = std::max(1, std::min({heads, 256 / units, a.rows >= 512 ? (heads + 3) / 4 : heads}));
    const int tokens = 256 / (units * slots);
    rope_vector_kernel<T, E><<<(unsigned)((a.rows + tokens - 1) / tokens), 256, 0, stream>>>(a, units, slots, tokens);
  } else if constexpr (E > 1) {
    return launch_rope_type<T, E / 2>(a, stream);
  } else {
    const int64_t total = a.rows * heads * (a.pairs + a.rest);
    rope_any_kernel<T><<<(unsigned)std::min<int64_t>((total + 255) / 256, 1 << 16), 256, 0, stream>>>(a);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rope_apply(const RopeAngles& angles, int type, const nemo_rope_heads& q, const nemo_rope_heads* k,
                             int64_t rows, const int64_t* positions, int64_t base, hipStream_t stream) {
  RopeArgs a{q, k ? *k : nemo_rope_heads{}, angles.turns, positions, base, rows, angles.magnitude, angles.head_dim,
             angles.rotary / 2, 0, angles.half};
  auto copied = [](const nemo_rope_heads& s) {
    return s.heads && !(s.x == s.y && s.x_row == s.y_row && s.x_head == s.y_head);
  };
  if (copied(a.q) || copied(a.k)) a.rest = angles.head_dim - angles.rotary;
  if (rows == 0 || a.q.heads + a.k.heads == 0) return hipSuccess;
  switch (type) {
    case NEMO_TYPE_F32: return launch_rope_type<float>(a, stream);
    case NEMO_TYPE_F16: return launch_rope_type<half_t>(a, stream);
    case NEMO_TYPE_BF16: return launch_rope_type<bf16_t>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace nemo
