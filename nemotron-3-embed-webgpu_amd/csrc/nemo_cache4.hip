// Rows into a paged cache of 4-bit floats, keys turned on the way, and out of
// it again, for gfx950 (include/nemo.h nemo_cache4_append, nemo_cache4_read).
//
// 32 values x of a head share the power of two 2^s, the smallest with max |x|
// <= 7 2^s, and become the nearest E2M1 float of x / 2^s. Next to a border
// between two codes the 32-bit roundings of a rotation decide wrongly a few
// times in a million values, so angles, rotation and the division by 2^s (exact)
// are in 64 bits, and the one rounding is that to the code.
//
// A wave takes a token. Lane l computes the angle of pair l, which the 16 lanes
// of a head pick up from LDS: lane l's head is l / 16 (of four at a time), its
// values D / 16 (l % 16) .., one 4-byte piece of codes for heads of 128.
#include <algorithm>

#include "nemo_cache4.h"

namespace nemo {

namespace {

struct RowsArgs {
  nemo_cache4_rows r;
  Cache4 c;
  RopeAngles angles;  // turns null: keys as they are
};

// A row's token of its request, none (-1) for rows before the first request and
// behind the last and for those before token 0, and the token's page, none (-1)
// for those that are not there. A wave looks at 64 requests at a time, evenly over
// those that it may be.
struct Token {
  int at, page;
  __device__ __forceinline__ Token(const Cache4& c, const int32_t* q_start, int64_t rows, int64_t t) {
    const int lane = threadIdx.x & 63;
    auto row = [&](int at) { return (int64_t)min((int64_t)max(q_start[at], 0), rows); };
    int from = 0, left = c.count;
    while (left > 64) {
      const int step = (left + 63) >> 6, i = from + min(lane * step, left - 1);
      const int n = (int)__popcll(__builtin_amdgcn_ballot_w64(lane * step < left && row(i) <= t));
      from += max(n - 1, 0) * step;
      left = min(step, c.count - from);
    }
    const int i = min(from + lane, c.count - 1);
    const int begin = (int)row(i), end = (int)row(i + 1), len = c.kv_len[i];
    const int n = (int)__popcll(__builtin_amdgcn_ballot_w64(lane < left && begin <= t));
    const int of = max(n - 1, 0);
    const int end_of = __builtin_amdgcn_readlane(end, of);
    const int64_t p = (int64_t)__builtin_amdgcn_readlane(len, of) - end_of + t;
    at = n == 0 || t >= end_of || p < 0 ? -1 : (int)p;
    page = -1;
    if (at >= 0 && at >> c.shift < c.table_row) page = c.table[(from + of) * c.table_row + (at >> c.shift)];
    if (page >= c.pages) page = -1;
  }
};

// The largest magnitude's bits of 32 values, of which a lane has those of `m`.
template <int LANES>
__device__ __forceinline__ uint64_t block_max(uint64_t m) {
#pragma unroll
  for (int o = 1; o < LANES; o *= 2) m = max(m, (uint64_t)__shfl_xor((unsigned long long)m, o, 64));
  return m;
}

// v in 32 bits, with its last bit set where they do not hold it, rounded to zero
// before: a code of that is v's own.
__device__ __forceinline__ float odd(double v) {
  const float f = (float)v;
  uint32_t bits = __float_as_uint(f);
  if ((double)f != v) bits = (bits - (fabs((double)f) > fabs(v) ? 1 : 0)) | 1;
  return __uint_as_float(bits);
}

// Codes of N values, two a byte, and the scale byte of the 32 that a lane's are
// part of.
template <int N>
__device__ __forceinline__ uint32_t encode(const double (&x)[N], int* scale) {
  uint64_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) m = max(m, __builtin_bit_cast(uint64_t, x[i]) & 0x7fffffffffffffffull);
  m = block_max<32 / N>(m);
  const int e = (int)(m >> 52);
  if (e == 0x7ff) {  // an infinity or a NaN
    *scale = 255;
    return 0;
  }
  // m = 2^(e - 1023) (1 + f): at most 7 2^s = 1.75 2^(s + 2)
  const int s = min(max(e - 1023 - 2 + ((m & 0xfffffffffffffull) > 0xc000000000000ull), -126), 125);
  *scale = s + 127;
  const double inv = __builtin_bit_cast(double, (uint64_t)(1023 - s) << 52);
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float a = odd(x[i] * inv), b = odd(x[i + 1] * inv);
    switch (i / 2) {
      case 0: codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, a, b, 1.0f, 0); break;
      case 1: codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, a, b, 1.0f, 1); break;
      case 2: codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, a, b, 1.0f, 2); break;
      default: codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, a, b, 1.0f, 3); break;
    }
  }
  return codes;
}

template <typename T, int D>
__global__ __launch_bounds__(256) void cache4_append_kernel(RowsArgs a) {
  typedef Cache4Head<D> Head;
  constexpr int N = D / 16;
  __shared__ double2 angles[4][64];  // cosine and sine
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = (int64_t)blockIdx.x * 4 + wave;
  if (t >= a.r.rows) return;  // (no barrier follows: a wave has its own angles)
  const Token token(a.c, a.r.q_start, a.r.rows, t);
  if (token.at < 0 || token.page < 0) return;
  const int in = token.at & ((1 << a.c.shift) - 1), n = lane & 15, pairs = a.angles.rotary / 2;
  const bool turn = a.angles.turns != nullptr, half = a.angles.half;
  if (turn) {
    if (lane < pairs) {
      double p = (double)(a.r.positions ? a.r.positions[t] : (int64_t)token.at) * a.angles.turns[lane];
      p -= rint(p);
      double s, c;
      sincospi(2.0 * p, &s, &c);
      angles[wave][lane] = make_double2(c * a.angles.magnitude, s * a.angles.magnitude);
    }
    __builtin_amdgcn_wave_barrier();
  }
  for (int h = lane >> 4; h < 2 * a.c.kv_heads; h += 4) {
    const bool value = h >= a.c.kv_heads;
    const int kvh = value ? h - a.c.kv_heads : h;
    const T* x = value ? (const T*)a.r.v + t * a.r.v_row + kvh * a.r.v_head
                       : (const T*)a.r.k + t * a.r.k_row + kvh * a.r.k_head;
    double v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (double)(float)x[N * n + i];
    if (!value && turn) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int d = N * n + i;
        if (d >= 2 * pairs) continue;
        const bool second = half ? d >= pairs : d & 1;
        const int pair = half ? (second ? d - pairs : d) : d >> 1;
        const double other = (double)(float)x[half ? (second ? d - pairs : d + pairs) : d ^ 1];
        const double2 cs = angles[wave][pair];
        v[i] = second ? other * cs.y + v[i] * cs.x : v[i] * cs.x - other * cs.y;
      }
    }
    int scale;
    const uint32_t codes = encode(v, &scale);
    uint8_t* const to = a.c.data + a.c.head<D>(token.page, kvh);
    uint8_t* const at = to + (value ? Head::v_codes(a.c.shift, in, n) : Head::k_codes(in) + n * Head::kScales);
    if constexpr (D == 128) *(uint32_t*)at = codes;
    else *(uint16_t*)at = (uint16_t)codes;
    if (n % (32 / N) == 0) to[Head::scale(a.c.shift, value, in, n / (32 / N))] = (uint8_t)scale;
  }
}

// Values of a lane's piece: N codes of one scale.
template <typename T, int D>
__global__ __launch_bounds__(256) void cache4_read_kernel(RowsArgs a) {
  typedef Cache4Head<D> Head;
  constexpr int N = D / 16;
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.r.rows) return;
  const Token token(a.c, a.r.q_start, a.r.rows, t);
  if (token.at < 0) return;
  const int in = token.at & ((1 << a.c.shift) - 1), n = lane & 15;
  for (int h = lane >> 4; h < 2 * a.c.kv_heads; h += 4) {
    const bool value = h >= a.c.kv_heads;
    const int kvh = value ? h - a.c.kv_heads : h;
    uint32_t codes = 0;
    int scale = 127;
    if (token.page >= 0) {
      const uint8_t* const from = a.c.data + a.c.head<D>(token.page, kvh);
      const uint8_t* const at = from + (value ? Head::v_codes(a.c.shift, in, n) : Head::k_codes(in) + n * Head::kScales);
      codes = D == 128 ? *(const uint32_t*)at : *(const uint16_t*)at;
      scale = from[Head::scale(a.c.shift, value, in, n / (32 / N))];
    }
    T* x = value ? (T*)a.r.v + t * a.r.v_row + kvh * a.r.v_head : (T*)a.r.k + t * a.r.k_row + kvh * a.r.k_head;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int code = codes >> (4 * i) & 15, e = code >> 1 & 3, f = code & 1;
      // 2^(e - 1) (1 + f / 2), or f / 2
      const float m = e ? (float)(2 + f) * (float)(1 << e) * 0.25f : 0.5f * f;
      const float p = scale == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(m, scale - 127);
      x[N * n + i] = (T)(code & 8 ? -p : p);
    }
  }
}

template <typename Launch>
hipError_t by_type(int type, int head_dim, Launch&& launch) {
  auto typed = [&](auto t) {
    if (head_dim == 64) launch(t, std::integral_constant<int, 64>{});
    else launch(t, std::integral_constant<int, 128>{});
  };
  if (type == NEMO_TYPE_F32) typed(float{});
  else if (type == NEMO_TYPE_F16) typed(half_t{});
  else typed(bf16_t{});
  return hipGetLastError();
}

}  // namespace

hipError_t launch_cache4_append(const nemo_cache4_config& c, const nemo_cache4_pages& p, const nemo_cache4_rows& r,
                                const RopeAngles* angles, hipStream_t stream) {
  if (p.count == 0 || r.rows == 0) return hipSuccess;
  const RowsArgs a{r, Cache4(c, p), angles ? *angles : RopeAngles{}};
  return by_type(r.type, c.head_dim, [&](auto t, auto d) {
    cache4_append_kernel<decltype(t), decltype(d)::value><<<(unsigned)((r.rows + 3) / 4), 256, 0, stream>>>(a);
  });
}

hipError_t launch_cache4_read(const nemo_cache4_config& c, const nemo_cache4_pages& p, const nemo_cache4_rows& r,
                              hipStream_t stream) {
  if (p.count == 0 || r.rows == 0) return hipSuccess;
  const RowsArgs a{r, Cache4(c, p), RopeAngles{}};
  return by_type(r.type, c.head_dim, [&](auto t, auto d) {
    cache4_read_kernel<decltype(t), decltype(d)::value><<<(unsigned)((r.rows + 3) / 4), 256, 0, stream>>>(a);
  });
}

}  // namespace nemo
