// Rows into a paged cache of 4-bit floats, keys turned on the way, and out of
// it again, for gfx950 (include/nemo.h nemo_cache4_append, nemo_cache4_read).
//
// 32 values x of a head share the power of two 2^s, the smallest with max |x|
// <= 7 2^s, and become the nearest E2M1 float of x / 2^s, which is exact in 32
// bits. A rotation is not: an angle's remainder and its sine in 32 bits, the
// factor and two products leave it some 10 2^-24 of |a| + |b| off, and next to a
// border between codes it is decided wrongly a few times in a million values.
// So both ends of 2^-20 around it are coded, and from the first heads on whose codes
// or powers differ the wave takes the token's rotation again in 64 bits, behind the
// others: beside them it held registers for all, and its sines were taken by all.
//
// Appending is bound by a wave's chain of loads before its first write (the requests'
// bounds, the table's page, while the first rows come) and between its turns: a wave
// waits for 63 % of its cycles, and the vector units work for half. 31846
// tokens of 8 KV heads of 128 f16, 165 MB of rows and codes, take 45 us (3.7 TB/s), and 31
// (5.3 TB/s) to read. On the way: in 64 bits throughout 103; bounds in 32 bits, the rare
// path among them 52; values to codes by one conversion, without a product 48; the
// token looked up while its rows are on their way 45. (Several tokens a wave, which
// share the lookup, took more registers than it returned.)
//
// A wave takes a token. Lane l computes the angle of pair l, which the 16 lanes
// of a head pick up from LDS: lane l's head is l / 16 (of four at a time), its
// values D / 16 (l % 16) .., one 4-byte piece of codes for heads of 128.
#include <algorithm>
#include <type_traits>

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
// those that it may be; what `meanwhile` loads is not waited for.
struct Token {
  int at, page;
  template <typename Meanwhile>
  __device__ __forceinline__ Token(const Cache4& c, const int32_t* q_start, int64_t rows, int64_t t,
                                   Meanwhile&& meanwhile) {
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
    const int starts = q_start[i], ends = q_start[i + 1], len = c.kv_len[i];
    __builtin_amdgcn_sched_barrier(0);
    meanwhile();
    __builtin_amdgcn_sched_barrier(0);
    auto cut = [&](int at) { return (int)min((int64_t)max(at, 0), rows); };
    const int begin = cut(starts), end = cut(ends);
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

// The largest bits of LANES lanes side by side.
template <int LANES>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  auto moved = [](uint32_t x, auto to) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, decltype(to)::value, 15, 15, false);
  };
  v = max(v, moved(v, std::integral_constant<int, 0xb1>{}));                           // neighbours
  v = max(v, moved(v, std::integral_constant<int, 0x4e>{}));                           // pairs of a quad
  if constexpr (LANES > 4) v = max(v, moved(v, std::integral_constant<int, 0x141>{}));  // quads of 8
  return v;
}
template <int LANES>
__device__ __forceinline__ uint64_t lanes_max(uint64_t v) {
#pragma unroll
  for (int o = 1; o < LANES; o *= 2) v = max(v, (uint64_t)__shfl_xor((unsigned long long)v, o, 64));
  return v;
}

// v in 32 bits, with its last bit set where they do not hold it, rounded to zero
// before: a code of that is v's own.
__device__ __forceinline__ float odd(double v) {
  const float f = (float)v;
  uint32_t bits = __float_as_uint(f);
  if ((double)f != v) bits = (bits - (fabs((double)f) > fabs(v) ? 1 : 0)) | 1;
  return __uint_as_float(bits);
}

// Codes of N values over the power of two `scale`, two a byte: one division and one
// rounding, from 16 and 32 bits alike.
template <int B>
__device__ __forceinline__ uint32_t code_pair(uint32_t c, float a, float b, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, a, b, scale, B);
}
template <int B>
__device__ __forceinline__ uint32_t code_pair(uint32_t c, half_t a, half_t b, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, half2v{a, b}, scale, B);
}
template <int B>
__device__ __forceinline__ uint32_t code_pair(uint32_t c, bf16_t a, bf16_t b, float scale) {
  typedef bf16_t pair __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair{a, b}, scale, B);
}
template <typename T, int N>
using Vec = T __attribute__((ext_vector_type(N)));
template <int N, typename V>
__device__ __forceinline__ uint32_t codes_of(const V& u, float scale) {
  uint32_t c = code_pair<1>(code_pair<0>(0u, u[0], u[1], scale), u[2], u[3], scale);
  if constexpr (N == 8) c = code_pair<3>(code_pair<2>(c, u[4], u[5], scale), u[6], u[7], scale);
  return c;
}

// The bits of the largest |value| in 32 bits; those of NaN are larger than any.
template <typename T, int N>
__device__ __forceinline__ uint32_t peak_of(const Vec<T, N>& x) {
  if constexpr (std::is_same<T, float>::value) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    return m;
  } else {
    const Vec<unsigned short, N> bits = __builtin_bit_cast(Vec<unsigned short, N>, x) & (unsigned short)0x7fff;
    Vec<unsigned short, 2> m = bits.xy;
#pragma unroll
    for (int i = 2; i < N; i += 2) m = __builtin_elementwise_max(m, Vec<unsigned short, 2>{bits[i], bits[i + 1]});
    return __float_as_uint((float)__builtin_bit_cast(T, m[0] > m[1] ? m[0] : m[1]));
  }
}

// s of 32 values whose largest has exponent e, biased by `bias`, and a fraction of
// 1.75 or less or more: 2^(e - bias) (1 + f) is at most 7 2^s = 1.75 2^(s + 2).
__device__ __forceinline__ int power_of(int e, int bias, bool more) { return min(max(e - bias - 2 + more, -126), 125); }
__device__ __forceinline__ float two_to(int s) { return __uint_as_float((uint32_t)(127 + s) << 23); }

template <typename T, int N>
__device__ __forceinline__ void load_piece(const T* x, Vec<T, N>& v) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = x[i];  // (one load: the card takes any address)
}

// How keys are turned: not; neighbouring pairs; halves of which a lane has values
// of one, their partners one vector; halves in any other way.
enum Turn { kPlain, kPairs, kHalves, kHalvesAny };

template <typename T, int D, Turn TURN>
__global__ __launch_bounds__(256) void cache4_append_kernel(RowsArgs a) {
  typedef Cache4Head<D> Head;
  constexpr int N = D / 16, LANES = 32 / N;
  __shared__ float2 angles[4][64];  // cosine and sine
  __shared__ double2 angles64[4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = (int64_t)blockIdx.x * 4 + wave;
  if (t >= a.r.rows) return;  // (no barrier follows: a wave has its own angles)
  const int n = lane & 15, pairs = TURN == kPlain ? 0 : a.angles.rotary / 2, heads = a.c.kv_heads;
  // Of value i of the lane's: whether it is turned, and if so, whether it is its pair's second and which
  // pair (else any).
  const int half = N * n >= pairs ? N * n - pairs : N * n;
  auto is_turned = [&](int i) { return N * n + (TURN == kPairs ? i & ~1 : TURN == kHalves ? 0 : i) < 2 * pairs; };
  auto second = [&](int i) { return TURN == kPairs ? i & 1 : N * n + (TURN == kHalves ? 0 : i) >= pairs; };
  auto pair_of = [&](int i) {
    return TURN == kPairs ? N / 2 * n + i / 2 : TURN == kHalves ? min(half, 64 - N) + i
                                                                : min(N * n + i - (second(i) ? pairs : 0), 63);
  };
  struct Piece {
    Vec<T, N> x, other;
  };
  // (Lanes past the last head load its values too, and write nothing.)
  auto load_key = [&](Piece& p, int h) {
    const T* x = (const T*)a.r.k + t * a.r.k_row + min(h, heads - 1) * a.r.k_head;
    load_piece<T, N>(x + N * n, p.x);
    if constexpr (TURN == kHalves) {
      load_piece<T, N>(x + (!is_turned(0) ? N * n : second(0) ? half : N * n + pairs), p.other);
    } else if constexpr (TURN == kHalvesAny) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int d = N * n + i;
        p.other[i] = x[!is_turned(i) ? d : second(i) ? d - pairs : d + pairs];
      }
    }
  };
  auto load_value = [&](Piece& p, int h) {
    load_piece<T, N>((const T*)a.r.v + t * a.r.v_row + min(h, heads - 1) * a.r.v_head + N * n, p.x);
  };
  Piece key, value, next;
  int h0 = 4 * blockIdx.y, h = h0 + (lane >> 4);
  double turns = 0;  // whole turns of pair `lane` a position, then at the token's, less the whole ones
  int64_t position = 0;
  if constexpr (TURN != kPlain) {
    turns = a.angles.turns[min(lane, pairs - 1)];
    if (a.r.positions) position = a.r.positions[t];
  }
  const Token token(a.c, a.r.q_start, a.r.rows, t, [&] {
    load_key(key, h);
    load_value(value, h);
  });
  if (token.at < 0 || token.page < 0) return;
  const int in = token.at & ((1 << a.c.shift) - 1);
  if constexpr (TURN != kPlain) {
    if (lane < pairs) {
      turns *= (double)(a.r.positions ? position : (int64_t)token.at);
      turns -= rint(turns);
      float s, c;
      sincospif(2.0f * (float)turns, &s, &c);
      angles[wave][lane] = make_float2(c * a.angles.magnitude, s * a.angles.magnitude);
    }
    __builtin_amdgcn_wave_barrier();
  }
  const int by = 4 * gridDim.y;
  uint8_t* to = a.c.data + a.c.head<D>(token.page, h);
  const int64_t step = a.c.head<D>(0, by);
  auto write = [&](bool is_value, uint32_t codes, int s, bool bad) {
    uint8_t* const at = to + (is_value ? Head::v_codes(a.c.shift, in, n) : Head::k_codes(in) + n * Head::kScales);
    if (bad) codes = 0;
    if constexpr (D == 128) *(uint32_t*)at = codes;
    else *(uint16_t*)at = (uint16_t)codes;
    if (n % LANES == 0) to[Head::scale(a.c.shift, is_value, in, n / LANES)] = bad ? 255 : (uint8_t)(s + 127);
  };
  auto power32 = [](uint32_t bits) { return power_of((int)(bits >> 23), 127, (bits & 0x7fffff) > 0x600000); };
  // Values as they are.
  auto plain = [&](const Piece& piece, bool is_value, bool real) {
    const uint32_t peak = lanes_max<LANES>(peak_of<T, N>(piece.x));
    const int s = power32(peak);
    const uint32_t codes = codes_of<N>(piece.x, two_to(s));
    if (real) write(is_value, codes, s, peak >= 0x7f800000u);
  };
  const float rel = fabsf(a.angles.magnitude) * 0x1p-20f;
  // In 32 bits; whether that is enough. `whole`: every value is turned.
  auto turned = [&](const Piece& piece, bool real, auto whole) {
    // `all`: at least any |a| + |b|, and not finite where a value is not
    float u[N], low[N], high[N], peak = 0.f, all = 0.f;
    asm volatile("" ::: "memory");  // read the angles here: for all heads they would take 2 N registers
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float own = (float)piece.x[i];
      const float other = (float)(TURN == kPairs ? piece.x[i ^ 1] : piece.other[i]);
      const float2 by = angles[wave][pair_of(i)];
      float most = fabsf(own) + fabsf(other), add = TURN == kPairs && i & 1 ? 0.f : most;
      u[i] = fmaf(other, second(i) ? by.y : -by.y, own * by.x);
      if (!decltype(whole)::value && !is_turned(i)) {
        most = 0.f;
        add = fabsf(own);
        u[i] = own;
      }
      all += add;
      peak = fmaxf(peak, fabsf(u[i]));
      low[i] = fmaf(-most, rel, u[i]);
      high[i] = fmaf(most, rel, u[i]);
    }
    peak = __uint_as_float(lanes_max<LANES>(__float_as_uint(peak)));
    all = __uint_as_float(lanes_max<LANES>(__float_as_uint(all)));
    const float error = all * rel;
    const int s = power32(__float_as_uint(peak));
    const uint32_t codes = codes_of<N>(low, two_to(s));
    if (real) write(false, codes, s, false);
    // (what is small enough to lose bits in 32 is taken again too)
    return codes == codes_of<N>(high, two_to(s)) && peak + error < INFINITY && !(peak < 0x1p-100f && all != 0.f) &&
           power32(__float_as_uint(fmaxf(peak - error, 0.f))) == power32(__float_as_uint(peak + error));
  };
  // (All lanes stay in the loops: a wave votes, and lanes exchange. Those past the last head write nothing.)
  int again = heads;  // where heads begin that 32 bits are not enough for
  for (; h0 < heads; h0 += by, h += by) {
    load_key(next, h + by);
    if constexpr (TURN == kPlain) {
      plain(key, false, h < heads);
    } else {
      const bool enough = 2 * pairs == D ? turned(key, h < heads, std::true_type{})
                                         : turned(key, h < heads, std::false_type{});
      if (__builtin_amdgcn_ballot_w64(!enough)) again = min(again, h0);
    }
    key = next;
    load_value(next, h + by);
    plain(value, true, h < heads);
    value = next;
    to += step;
  }
  if constexpr (TURN != kPlain) {
    if (again >= heads) return;
    asm volatile("" : "+v"(turns));  // keeps the rare path's sines off the others' way
    if (lane < pairs) {
      double s, c;
      sincospi(2.0 * turns, &s, &c);
      angles64[wave][lane] = make_double2(c * a.angles.magnitude, s * a.angles.magnitude);
    }
    __builtin_amdgcn_wave_barrier();
    h = again + (lane >> 4);
    to = a.c.data + a.c.head<D>(token.page, h);
    for (h0 = again; h0 < heads; h0 += by, h += by, to += step) {
      load_key(key, h);
      double v[N];
      uint64_t m = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        asm volatile("" ::: "memory");  // one by one: fewer registers
        const double own = (double)(float)key.x[i];
        v[i] = own;
        if (is_turned(i)) {
          const double other = (double)(float)(TURN == kPairs ? key.x[i ^ 1] : key.other[i]);
          const double2 cs = angles64[wave][pair_of(i)];
          v[i] = fma(other, second(i) ? cs.y : -cs.y, own * cs.x);
        }
        m = max(m, __builtin_bit_cast(uint64_t, v[i]) & 0x7fffffffffffffffull);
      }
      m = lanes_max<LANES>(m);
      const int s = power_of((int)(m >> 52), 1023, (m & 0xfffffffffffffull) > 0xc000000000000ull);
      const double inv = __builtin_bit_cast(double, (uint64_t)(1023 - s) << 52);
      float u[N];
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = odd(v[i] * inv);
      if (h < heads) write(false, codes_of<N>(u, 1.f), s, m >= 0x7ff0000000000000ull);
    }
  }
}

// Pairs of values by the conversions from 4 bits.
template <typename T, int B>
__device__ __forceinline__ void decode(uint32_t codes, float scale, T& a, T& b) {
  if constexpr (std::is_same<T, float>::value) {
    const float2v v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, B);
    a = v[0], b = v[1];
  } else if constexpr (std::is_same<T, half_t>::value) {
    const half2v v = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, B);
    a = v[0], b = v[1];
  } else {
    const auto v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B);
    a = v[0], b = v[1];
  }
}

template <typename T, int D>
__global__ __launch_bounds__(256) void cache4_read_kernel(RowsArgs a) {
  typedef Cache4Head<D> Head;
  constexpr int N = D / 16;
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.r.rows) return;
  const Token token(a.c, a.r.q_start, a.r.rows, t, [] {});
  if (token.at < 0) return;
  const int in = token.at & ((1 << a.c.shift) - 1), n = lane & 15;
#pragma unroll 2
  for (int h = 4 * blockIdx.y + (lane >> 4); h < 2 * a.c.kv_heads; h += 4 * gridDim.y) {
    const bool value = h >= a.c.kv_heads;
    const int kvh = value ? h - a.c.kv_heads : h;
    uint32_t codes = 0, scale = 127;
    if (token.page >= 0) {
      const uint8_t* const from = a.c.data + a.c.head<D>(token.page, kvh);
      const uint8_t* const at = from + (value ? Head::v_codes(a.c.shift, in, n) : Head::k_codes(in) + n * Head::kScales);
      codes = D == 128 ? *(const uint32_t*)at : *(const uint16_t*)at;
      scale = from[Head::scale(a.c.shift, value, in, n / (32 / N))];
    }
    const float power = __uint_as_float(scale << 23);
    T v[N];
    decode<T, 0>(codes, power, v[0], v[1]);
    decode<T, 1>(codes, power, v[2], v[3]);
    if constexpr (N == 8) {
      decode<T, 2>(codes, power, v[4], v[5]);
      decode<T, 3>(codes, power, v[6], v[7]);
    }
    T* x = (value ? (T*)a.r.v + t * a.r.v_row + kvh * a.r.v_head : (T*)a.r.k + t * a.r.k_row + kvh * a.r.k_head) + N * n;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = v[i];  // (one store, as load_piece)
  }
}

// Waves of a token: one, but for few tokens one for every 4 of `heads` heads (64 tokens of 8 KV
// heads of 128: append 4.5 us, read 2.7; by one wave each 5.7 and 3.6).
dim3 grid_of(int64_t rows, int heads) {
  return dim3((unsigned)((rows + 3) / 4), rows <= 1024 ? std::min((heads + 3) / 4, 64) : 1);
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
    const dim3 grid = grid_of(r.rows, c.kv_heads);
    typedef decltype(t) T;
    constexpr int D = decltype(d)::value;
    if (!angles) cache4_append_kernel<T, D, kPlain><<<grid, 256, 0, stream>>>(a);
    else if (!angles->half) cache4_append_kernel<T, D, kPairs><<<grid, 256, 0, stream>>>(a);
    else if (angles->rotary / 2 % (D / 16) == 0) cache4_append_kernel<T, D, kHalves><<<grid, 256, 0, stream>>>(a);
    else cache4_append_kernel<T, D, kHalvesAny><<<grid, 256, 0, stream>>>(a);
  });
}

hipError_t launch_cache4_read(const nemo_cache4_config& c, const nemo_cache4_pages& p, const nemo_cache4_rows& r,
                              hipStream_t stream) {
  if (p.count == 0 || r.rows == 0) return hipSuccess;
  const RowsArgs a{r, Cache4(c, p), RopeAngles{}};
  return by_type(r.type, c.head_dim, [&](auto t, auto d) {
    cache4_read_kernel<decltype(t), decltype(d)::value><<<grid_of(r.rows, 2 * c.kv_heads), 256, 0, stream>>>(a);
  });
}

}  // namespace nemo
