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
#include <type_traits>

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

// ---------------------------------------------------------------------------
// The norm of each head on the way: h = x / sqrt(mean x^2 + eps) w, then turned.
// A head is `lanes` lanes of a wave, each with NI items of it: by halves the
// vectors of a pair's first and second values (two vectors side by side behind
// the pairs), interleaved one vector. The lanes add up their squares, so a
// head is read once, and a thread's angles and weights serve every `slots`-th
// head of its token.
// ---------------------------------------------------------------------------

// E values, read and written as one vector where the addresses allow it.
template <typename T, int E, bool VECTORS>
struct Values {
  typedef T vec __attribute__((ext_vector_type(E)));
  vec v;
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VECTORS) {
      v = *(const vec*)p;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = p[e];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (VECTORS) {
      *(vec*)p = v;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) p[e] = v[e];
    }
  }
};

// The sum over `lanes` (a power of two) lanes side by side.
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  auto moved = [](float x, auto to) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), decltype(to)::value, 15, 15, false));
  };
  if (lanes > 1) v += moved(v, std::integral_constant<int, 0xb1>{});   // neighbours
  if (lanes > 2) v += moved(v, std::integral_constant<int, 0x4e>{});   // pairs of a quad
  if (lanes > 4) v += moved(v, std::integral_constant<int, 0x141>{});  // quads of 8, mirrored
  if (lanes > 8) v += moved(v, std::integral_constant<int, 0x140>{});  // halves of 16, mirrored
  if (lanes > 16) v += __shfl_xor(v, 16, 64);
  if (lanes > 32) v += __shfl_xor(v, 32, 64);
  return v;
}

template <typename T, int E, bool HALF, bool VECTORS, int NI>
__global__ __launch_bounds__(256) void rope_norm_kernel(RopeArgs a, nemo_head_norm n, int lanes, int slots,
                                                        int tokens) {
  constexpr int V = HALF ? 2 : 1, C = HALF ? E : E / 2;  // vectors and pairs of an item
  const int per = lanes * slots, l = threadIdx.x % lanes;
  const int64_t t = (int64_t)blockIdx.x * tokens + threadIdx.x / per;
  if ((int)threadIdx.x >= tokens * per || t >= a.rows) return;  // (a head's lanes together)
  const int slot = blockIdx.y * slots + threadIdx.x % per / lanes;
  slots *= gridDim.y;
  const int items = a.head_dim / (V * E);
  int at[NI][V];
  bool real[NI], turned[NI];
  float2 cs[NI][C];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int item = l + lanes * i;
    real[i] = item < items;
    turned[i] = real[i] && (HALF ? item < a.pairs / E : item < 2 * a.pairs / E);
    at[i][0] = HALF && !turned[i] ? 2 * E * item : E * item;  // (2 pairs + 2 E (item - pairs / E))
    if constexpr (HALF) at[i][1] = turned[i] ? a.pairs + E * item : at[i][0] + E;
    if (!real[i]) {
#pragma unroll
      for (int v = 0; v < V; ++v) at[i][v] = 0;
    }
  }
  bool angles = false;
  const float inv = 1.0f / a.head_dim;
  typedef Values<T, E, VECTORS> vec;
  // Every `slots`-th head of q or k from `first` on; the next one's values are on their way.
  auto turn = [&](const nemo_rope_heads& s, const float* weight, int64_t weight_head, int first) {
    if (first >= s.heads) return;
    const T* x = (const T*)s.x + t * s.x_row + first * s.x_head;
    T* y = (T*)s.y + t * s.y_row + first * s.y_head;
    vec now[NI][V], next[NI][V];
    auto load = [&](vec (&to)[NI][V]) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) to[i][v].load(x + at[i][v]);
    };
    load(now);
    float w[NI][V][E];
    auto weights = [&](int h) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int e = 0; e < E; ++e) w[i][v][e] = weight ? weight[h * weight_head + at[i][v] + e] : 1.f;
    };
    weights(first);
    if (!angles) {
      const double p = rope_position(a, t);
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int c = 0; c < C; ++c)
          cs[i][c] = turned[i] ? rope_angle(a, C * (l + lanes * i) + c, p) : make_float2(1.f, 0.f);
      angles = true;
    }
    for (int h = first; h < s.heads; h += slots) {
      if (h + slots < s.heads) {
        x += slots * s.x_head;
        load(next);
      }
      float r[NI][V][E], sum = 0.f;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int e = 0; e < E; ++e) {
            r[i][v][e] = real[i] ? (float)now[i][v].v[e] : 0.f;
            sum = fmaf(r[i][v][e], r[i][v][e], sum);
          }
      const float mean = fmaf(lanes_sum(sum, lanes), inv, n.epsilon);
      const float f = mean >= 0x1p-100f ? __builtin_amdgcn_rsqf(mean) : 1.0f / sqrtf(mean);  // (rsq of small ones is 0)
      if (weight_head && h > first) weights(h);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int e = 0; e < E; ++e) r[i][v][e] *= f * w[i][v][e];
        if (turned[i]) {
#pragma unroll
          for (int c = 0; c < C; ++c) {
            float& u = HALF ? r[i][0][c] : r[i][0][2 * c];
            float& z = HALF ? r[i][V - 1][c] : r[i][0][2 * c + 1];
            const float turned_u = u * cs[i][c].x - z * cs[i][c].y;
            z = u * cs[i][c].y + z * cs[i][c].x;
            u = turned_u;
          }
        }
        if (!real[i]) continue;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          vec out;
#pragma unroll
          for (int e = 0; e < E; ++e) out.v[e] = (T)r[i][v][e];
          out.store(y + at[i][v]);
        }
      }
      y += slots * s.y_head;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) now[i][v] = next[i][v];
    }
  };
  turn(a.q, n.q_weight, n.q_weight_head, slot);
  // head h of both is slot h % slots'
  const int passed = a.q.heads % slots;
  turn(a.k, n.k_weight, n.k_weight_head, slot >= passed ? slot - passed : slot - passed + slots);
}

// By the widest vectors that sizes, strides and addresses allow.
template <typename T, int E = 16 / sizeof(T)>
hipError_t launch_rope_norm_type(const RopeArgs& a, const nemo_head_norm& n, hipStream_t stream) {
  const int heads = a.q.heads + a.k.heads, rest = a.head_dim - 2 * a.pairs, bytes = E * sizeof(T);
  const bool fits = a.half ? a.pairs % E == 0 && rest % (2 * E) == 0
                           : E > 1 && 2 * a.pairs % E == 0 && a.head_dim % E == 0;
  const bool vectors = aligned_heads(a.q, E, bytes) && (!a.k.heads || aligned_heads(a.k, E, bytes));
  auto launch = [&](auto half, auto v, auto ni, int items) {
    int lanes = 1;
    while (lanes < items && lanes < 64) lanes *= 2;
    // As many heads a thread as leave the chip 8 waves a SIMD.
    const int64_t want = (1 << 19) / (a.rows * lanes) + 1;
    const int all = (int)std::min<int64_t>(heads, want), slots = std::min(all, 256 / lanes);
    const int tokens = 256 / (lanes * slots), parts = (all + slots - 1) / slots;
    rope_norm_kernel<T, E, decltype(half)::value, decltype(v)::value, decltype(ni)::value>
        <<<dim3((unsigned)((a.rows + tokens - 1) / tokens), parts), 256, 0, stream>>>(a, n, lanes, slots, tokens);
    return hipGetLastError();
  };
  auto sized = [&](auto half, auto v) {
    const int items = a.head_dim / (decltype(half)::value ? 2 * E : E);
    if (items <= 64) return launch(half, v, std::integral_constant<int, 1>{}, items);
    if (items <= 128) return launch(half, v, std::integral_constant<int, 2>{}, items);
    if constexpr (E <= 4) {
      if (items <= 256) return launch(half, v, std::integral_constant<int, 4>{}, items);
      if constexpr (E <= 2) return launch(half, v, std::integral_constant<int, 8>{}, items);
    }
    return hipErrorInvalidValue;  // (1024 values are 128 items of 8, 256 of 4, 512 of 2)
  };
  if (fits && vectors) {
    if constexpr (E > 1) {
      if (!a.half) return sized(std::false_type{}, std::true_type{});
    }
    if (a.half) return sized(std::true_type{}, std::true_type{});
  }
  if constexpr (E == 2) {  // single values
    if (!a.half) return sized(std::false_type{}, std::false_type{});
  }
  if constexpr (E > 1) return launch_rope_norm_type<T, E / 2>(a, n, stream);
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_rope_norm(const RopeAngles& angles, int type, const nemo_rope_heads& q, const nemo_rope_heads* k,
                            const nemo_head_norm& norm, int64_t rows, const int64_t* positions, int64_t base,
                            hipStream_t stream) {
  const RopeArgs a{q, k ? *k : nemo_rope_heads{}, angles.turns, positions, base, rows, angles.magnitude,
                   angles.head_dim, angles.rotary / 2, 0, angles.half};
  if (rows == 0 || a.q.heads + a.k.heads == 0) return hipSuccess;
  switch (type) {
    case NEMO_TYPE_F32: return launch_rope_norm_type<float>(a, norm, stream);
    case NEMO_TYPE_F16: return launch_rope_norm_type<half_t>(a, norm, stream);
    case NEMO_TYPE_BF16: return launch_rope_norm_type<bf16_t>(a, norm, stream);
    default: return hipErrorInvalidValue;
  }
}

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
