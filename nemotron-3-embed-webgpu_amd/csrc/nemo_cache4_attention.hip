// Attention over a paged cache of 4-bit floats for gfx950 (include/nemo.h
// nemo_cache4_attention): softmax(scale q.k) v over the keys j <= p + right that
// have j >= p - left or j < sinks.
//
// Rows are (query, head of the group) pairs of one request and KV head, query
// by query; a wave takes 16 QT of them and 32 keys a step. Codes go from memory
// to registers and become 16-bit floats there, two by an instruction and
// exactly: no LDS, no scale left to be applied.
//
// Scores are taken transposed, S^T = K Q^T (two tiles of 16 keys x 16 rows by
// v_mfma_f32_16x16x32), so a lane holds one row, and which keys a tile has is
// free: lane group h = lane / 16 gets the scores of keys 8 h .. 8 h + 7, in order,
// as its registers of both tiles. That is the second operand of O^T = V^T P^T
// (16 columns x 16 rows over 32 keys). K's operand is a key's D / 4 values from
// D / 4 h on, 16 bytes for heads of 128; V's operand is one column of 8 keys: a
// lane decodes D / 16 columns of its 8 keys, which lie side by side in the cache,
// and exchanges halves of neighbouring keys' registers.
#include <algorithm>
#include <type_traits>

#include "nemo_attention_tile.h"
#include "nemo_cache4.h"
#include "nemo_lds_copy.h"

namespace nemo {

namespace {

struct AttendArgs {
  nemo_cache4_queries b;
  Cache4 c;
  int group, left, right, sinks;
  float scale2;  // of the scores, in units of log2
  // row / group for rows below 2^31: (row + the high half of row * magic) >> shift
  uint32_t magic;
  int shift;
  __device__ __forceinline__ int query(int row) const {
    return (int)((__umulhi((uint32_t)row, magic) + (uint32_t)row) >> shift);
  }
};

// The window of a query at p over a request's n keys: [lo, hi).
struct Seen {
  int lo, hi;
  __device__ __forceinline__ Seen(int from, int to) : lo(from), hi(to) {}
  __device__ __forceinline__ Seen(const AttendArgs& a, int p, int n) {
    hi = max(0, min(n, a.right >= kUnbounded ? n : p + a.right + 1));
    lo = a.left >= kUnbounded ? 0 : min(hi, max(0, p - a.left));
  }
};

// The request of tile number t, and the number of its first tile; tiles of ROWS
// (query, head of the group) rows are numbered through a batch without a
// table: request i's first number is floor(q_start[i] group / ROWS) + i, which
// leaves it at least as many numbers as it has tiles. None (i = -1) before the
// first request. A wave looks at 64 requests at a time, evenly over those that
// it may be.
struct Request {
  int i, tile, q0, queries, behind, keys;  // behind: position of query 0; keys: tokens that the table has room for
  __device__ __forceinline__ Request(const AttendArgs& a, int t, int ROWS) {
    const int lane = threadIdx.x & 63;
    auto row = [&](int at) { return min(max(a.b.q_start[at], 0), (int)a.b.q_rows); };
    auto number = [&](int begin, int at) { return (int)((int64_t)begin * a.group / ROWS) + at; };
    int from = 0, left = a.c.count;
    while (left > 64) {
      const int step = (left + 63) >> 6, at = from + min(lane * step, left - 1);
      const int n = (int)__popcll(__builtin_amdgcn_ballot_w64(lane * step < left && number(row(at), at) <= t));
      from += max(n - 1, 0) * step;
      left = min(step, a.c.count - from);
    }
    const int at = min(from + lane, a.c.count - 1), begin = row(at), end = row(at + 1);
    const int len = min(max(a.c.kv_len[at], 0), 1 << 30);
    const int first = number(begin, at);
    const int n = (int)__popcll(__builtin_amdgcn_ballot_w64(lane < left && first <= t));
    i = from + n - 1;
    if (!n) i = -1;
    const int of = max(n - 1, 0);
    tile = __builtin_amdgcn_readlane(first, of);
    q0 = __builtin_amdgcn_readlane(begin, of);
    queries = max(__builtin_amdgcn_readlane(end, of) - q0, 0);
    const int tokens = __builtin_amdgcn_readlane(len, of);
    behind = tokens - queries;
    keys = (int)min((int64_t)tokens, a.c.table_row << a.c.shift);
  }
};

// The blocks of 32 keys that the rows of queries at p0 .. p1 see: those of the
// sinks before the window, then the window's.
struct Blocks {
  int sinks, skip, n;
  __device__ __forceinline__ Blocks(const AttendArgs& a, const Seen& first, const Seen& last) {
    const int lo = first.lo >> 5, hi = (last.hi + 31) >> 5;
    sinks = min((min(a.sinks, last.hi) + 31) >> 5, lo);
    skip = lo - sinks;
    n = max(hi - skip, 0);
  }
  __device__ __forceinline__ int block(int t) const { return t < sinks ? t : t + skip; }
};

template <typename T>
struct Mma16;
template <>
struct Mma16<half_t> {
  typedef half8v frag;
  typedef half2v pair;
  static constexpr int kFinite = 140;  // largest scale byte under which every code is finite
  static constexpr uint32_t kExponent = 0x7c00, kOne = 0x3c00;
  static __device__ __forceinline__ float add(pair p, float sum) {
    return __builtin_amdgcn_fdot2(p, pair{(half_t)1.f, (half_t)1.f}, sum, false);
  }
  static __device__ __forceinline__ float4v mma(frag a, frag b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  template <int B>
  static __device__ __forceinline__ uint32_t decode(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, B));
  }
};
template <>
struct Mma16<bf16_t> {
  typedef bf16_t frag __attribute__((ext_vector_type(8)));
  typedef bf16_t pair __attribute__((ext_vector_type(2)));
  static constexpr int kFinite = 252;
  static constexpr uint32_t kExponent = 0x7f80, kOne = 0x3f80;
  static __device__ __forceinline__ float add(pair p, float sum) {
    return __builtin_amdgcn_fdot2_f32_bf16(p, pair{(bf16_t)1.f, (bf16_t)1.f}, sum, false);
  }
  static __device__ __forceinline__ float4v mma(frag a, frag b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  template <int B>
  static __device__ __forceinline__ uint32_t decode(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B));
  }
};

// The power of two of byte i of eight scale bytes. (A conversion reads the
// exponent's bits alone, so those of other bytes beside it may stay.)
__device__ __forceinline__ float power(u32x2 bytes, int i) {
  const uint32_t w = bytes[i >> 2];
  const int s = 23 - 8 * (i & 3);
  return __uint_as_float(s >= 0 ? w << s : w >> -s);
}

// What a lane has of a block of 32 keys. K tile u's row l % 16 = 4 b + j is key
// 8 b + 4 u + j, so a lane's scores of both tiles are of keys that follow each other.
template <int D>
struct Raw {
  static constexpr int W = D / 32;  // registers of 8 codes: a key's quarter of K, 4 keys' pieces of V times two
  typedef uint32_t vec __attribute__((ext_vector_type(W)));
  vec k[2], v[2];
  u32x2 k_scales, v_scales;
  // The page's KV head begins at `head`; key t of it is the block's first.
  __device__ __forceinline__ void load(const uint8_t* head, int shift, int t, int lane) {
    typedef Cache4Head<D> Head;
    const int row = lane & 15, h = lane >> 4, key = 8 * (row >> 2) + (row & 3);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      k[u] = *(const vec*)(head + Head::k_codes(t + key + 4 * u) + h * (D / 8));
      v[u] = *(const vec*)(head + Head::v_codes(shift, t + 8 * h + 4 * u, row));
    }
    k_scales = *(const u32x2*)(head + Head::scale(shift, false, t + 8 * (row >> 2), h * (D / 32) / 4));
    v_scales = *(const u32x2*)(head + Head::scale(shift, true, t + 8 * h, row * (D / 32) / 16));
  }
};

// A wave's 16 QT rows: row 16 i + l % 16 in lane l for each i, whose group h = l / 16
// holds output columns D / 16 (4 h + e) + t in register e of o[i][t], and the sum
// of its own keys' probabilities.
template <typename T, int D, int QT>
struct Rows16 {
  static constexpr int W = D / 32, C = D / 16;
  typedef Mma16<T> M;
  typedef typename M::frag frag;
  typedef typename M::pair pair;
  // Queries: in registers for one tile of rows, else an LDS image of rows, 16-byte
  // chunk c of row r at c ^ (r % (D / 8)).
  static constexpr bool IMAGE = QT > 1;
  frag held[IMAGE ? 1 : W];
  const uint8_t* image;
  __device__ __forceinline__ frag query(int i, int w, int lane) const {
    if constexpr (!IMAGE) return held[w];
    const int row = lane & 15, chunk = W * (lane >> 4) + w;
    return *(const frag*)(image + (16 * i + row) * 2 * D + 16 * (chunk ^ (row & (D / 8 - 1))));
  }
  float4v o[QT][C];
  float m[QT], l[QT];  // reference and sum of the probabilities

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int t = 0; t < C; ++t) o[i][t] = float4v{0.f, 0.f, 0.f, 0.f};
    }
  }
  // Probabilities are taken against a reference that is raised when the sum of a
  // lane's 8 passes MOST, as in window attention: f16's largest is 2^BELOW and
  // more, so that what lies far below it keeps its share among f16's smallest
  // values.
  //
  // Sums of bf16's largest values leave 32 bits that way: a row whose sums do is
  // taken again 2^42 lower, where the probabilities of 2^30 keys add up to 1 at
  // most. Only such a row, since probabilities end 2^42 earlier too.
  static constexpr bool HALF = std::is_same<T, half_t>::value;
  float low[QT];  // by how much in units of log2, CAREFUL
  static __device__ __forceinline__ float exponentials(const float (&s)[8], float scale2, float m, frag& p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = (T)__builtin_amdgcn_exp2f(fmaf(s[i], scale2, -m));
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) v = M::add(pair{p[i], p[i + 1]}, v);
    return v;
  }
  template <bool CAREFUL>
  __device__ __forceinline__ void settle(int i, const float (&s)[8], float scale2, frag& p) {
    const bool lower = CAREFUL && !HALF && low[i] > 0.f;
    const float below = HALF ? 8.f : lower ? -low[i] : 0.f, most = HALF ? 0x1p20f : lower ? 0x1p-27f : 0x1p15f;
    float add = exponentials(s, scale2, m[i], p);
    if (__builtin_amdgcn_ballot_w64(!(add <= most))) {
      asm volatile("");  // keeps the rare path a branch
      float top = s[0];
#pragma unroll
      for (int r = 1; r < 8; ++r) top = fmaxf(top, s[r]);
      top *= scale2;
      int raise = !(add <= most);
#pragma unroll
      for (int x = 16; x < 64; x *= 2) {
        raise |= __shfl_xor(raise, x, 64);  // only the rows that ask: none depends on another
        top = fmaxf(top, __shfl_xor(top, x, 64));
      }
      const float raised = raise ? fmaxf(m[i], top - below) : m[i];
      const float alpha = m[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[i] - raised);
      l[i] *= alpha;
#pragma unroll
      for (int t = 0; t < C; ++t) o[i][t] *= alpha;
      m[i] = raised;
      add = exponentials(s, scale2, raised == -INFINITY ? 0.f : raised, p);
    }
    l[i] += add;
  }
  // Whether a value of the wave's rows is not finite, and how much lower each row is taken
  // again then.
  __device__ __forceinline__ bool spoilt(int lane) {
    uint64_t any = 0;
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      float z = l[i] * 0.f;
#pragma unroll
      for (int t = 0; t < C; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) z = fmaf(o[i][t][e], 0.f, z);
      const uint64_t lanes = __builtin_amdgcn_ballot_w64(z != 0.f);
      low[i] = lanes >> (lane & 15) & 0x0001000100010001ull ? 42.f : 0.f;  // (a row's four)
      any |= lanes;
    }
    return any != 0;
  }
};

// Which of the 8 keys from j on a row sees, as bits.
__device__ __forceinline__ uint32_t seen8(int j, const Seen& s, int sinks) {
  auto below = [&](int t) { return (1u << max(0, min(t - j, 8))) - 1; };
  return below(s.hi) & (~below(s.lo) | below(sinks));
}

// Takes out of a block what its V holds that is not finite: the rows that see such a
// value become NaN in its column, and its code is zero afterwards. Under a large scale
// byte smaller codes are finite, but for byte 255.
template <typename T, int D, int QT>
__device__ __forceinline__ void take_out(Rows16<T, D, QT>& a, Raw<D>& raw, bool hide, const uint32_t (&seen)[QT],
                                         uint32_t any) {
  typedef Mma16<T> M;
  typedef typename M::frag frag;
  auto byte = [&](int e) { return (int)(raw.v_scales[e >> 2] >> (8 * (e & 3)) & 255); };
  bool above = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) above |= byte(e) > M::kFinite && any >> e & 1;
  if (!__builtin_amdgcn_ballot_w64(above)) return;
  // Columns 2 b, 2 b + 1 of the lane's piece: byte b of a key's codes, D / 32 bytes.
  auto columns = [&](auto at) {
    constexpr int B = decltype(at)::value;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      asm volatile("" : "+v"(raw.v_scales[0]), "+v"(raw.v_scales[1]));  // nothing is kept from one to the next
      u32x4 bad = {0, 0, 0, 0};  // ones in the places of such values
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        constexpr int b[2] = {B, D == 128 ? B : B + 2};
        const int word = D == 128 ? e & 3 : e >> 1 & 1;
        const uint32_t codes = raw.v[e >> 2][word];
        const uint32_t pair = e & 1 ? M::template decode<b[1]>(codes, power(raw.v_scales, e))
                                    : M::template decode<b[0]>(codes, power(raw.v_scales, e));
        if (!(any >> e & 1) || (pair >> (16 * half) & M::kExponent) != M::kExponent) continue;
        bad[e >> 1] |= M::kOne << (16 * (e & 1));
        raw.v[e >> 2][word] = codes & ~(15u << (8 * b[e & 1] + 4 * half));
      }
#pragma unroll
      for (int i = 0; i < QT; ++i) {
        frag sees;
#pragma unroll
        for (int e = 0; e < 8; ++e) sees[e] = (T)(!hide || (seen[i] >> e & 1) ? 1.f : 0.f);
        const float4v n = M::mma(__builtin_bit_cast(frag, bad), sees, float4v{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n[e] > 0.f) a.o[i][2 * B + half][e] = __uint_as_float(0x7fc00000u);
      }
    }
  };
  columns(std::integral_constant<int, 0>{});
  columns(std::integral_constant<int, 1>{});
  if constexpr (D == 128) {
    columns(std::integral_constant<int, 2>{});
    columns(std::integral_constant<int, 3>{});
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (byte(e) == 255) raw.v_scales[e >> 2] &= ~(255u << (8 * (e & 3)));
}

// One block of 32 keys from key j0 on. `hide`: not every row sees all of them;
// `seen`: what its lane's rows see, `any`: what some row of the tile sees. CAREFUL: V's values
// that are not finite are taken out first and reach the rows that see them alone.
template <bool CAREFUL, typename T, int D, int QT>
__device__ __forceinline__ void attend(Rows16<T, D, QT>& a, Raw<D>& raw, float scale2, bool hide,
                                       const uint32_t (&seen)[QT], uint32_t any) {
  constexpr int W = D / 32;
  typedef Mma16<T> M;
  typedef typename M::frag frag;
  const int lane = threadIdx.x & 63;
  if constexpr (CAREFUL) take_out(a, raw, hide, seen, any);
  float4v s[QT][2];
  const float powers[2] = {__uint_as_float((raw.k_scales[0] >> (8 * (lane & 3))) << 23),
                           __uint_as_float((raw.k_scales[1] >> (8 * (lane & 3))) << 23)};
#pragma unroll
  for (int w = 0; w < W; ++w) {
    frag q[QT];
#pragma unroll
    for (int i = 0; i < QT; ++i) q[i] = a.query(i, w, lane);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t c = raw.k[u][w];
      const float power = powers[u];
      const u32x4 f = {M::template decode<0>(c, power), M::template decode<1>(c, power),
                       M::template decode<2>(c, power), M::template decode<3>(c, power)};
#pragma unroll
      for (int i = 0; i < QT; ++i)
        s[i][u] = M::mma(__builtin_bit_cast(frag, f), q[i], w ? s[i][u] : float4v{0.f, 0.f, 0.f, 0.f});
    }
  }
  frag p[QT];
  u32x2 scales = raw.v_scales;
  if (hide) {
    // values of keys that no row sees are taken times 2^-127
    uint32_t keep[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      keep[x] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) keep[x] |= any >> (4 * x + e) & 1 ? 255u << (8 * e) : 0;
      scales[x] &= keep[x];
    }
  }
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = s[i][e >> 2][e & 3];
    if (hide) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = seen[i] >> e & 1 ? v[e] : -INFINITY;
    }
    a.template settle<CAREFUL>(i, v, scale2, p[i]);
  }
  // V: columns 2 b, 2 b + 1 of the lane's piece, for each of its 8 keys in one register
  float power[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) power[e] = nemo::power(scales, e);
  auto columns = [&](auto at) {
    constexpr int B = decltype(at)::value;
    uint32_t r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (D == 128) r[e] = M::template decode<B>(raw.v[e >> 2][e & 3], power[e]);
      else r[e] = e & 1 ? M::template decode<B + 2>(raw.v[e >> 2][e >> 1 & 1], power[e])
                        : M::template decode<B>(raw.v[e >> 2][e >> 1 & 1], power[e]);
    }
    u32x4 low, high;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      low[e] = __builtin_amdgcn_perm(r[2 * e + 1], r[2 * e], 0x05040100u);
      high[e] = __builtin_amdgcn_perm(r[2 * e + 1], r[2 * e], 0x07060302u);
    }
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      a.o[i][2 * B] = M::mma(__builtin_bit_cast(frag, low), p[i], a.o[i][2 * B]);
      a.o[i][2 * B + 1] = M::mma(__builtin_bit_cast(frag, high), p[i], a.o[i][2 * B + 1]);
    }
  };
  columns(std::integral_constant<int, 0>{});
  columns(std::integral_constant<int, 1>{});
  if constexpr (D == 128) {
    columns(std::integral_constant<int, 2>{});
    columns(std::integral_constant<int, 3>{});
  }
}

// The rows over every `stride`-th block from `from` to before `end`. first, last: the
// windows of the rows' first and last query; lo, hi: those of the lane's rows.
template <bool CAREFUL, typename T, int D, int QT>
__device__ __forceinline__ void attend_blocks(const AttendArgs& a, Rows16<T, D, QT>& acc, const Request& r,
                                              const Blocks& blocks, const Seen& first, const Seen& last,
                                              const int (&lo)[QT], const int (&hi)[QT], int kvh, int from, int stride,
                                              int end) {
  acc.clear();
  const int steps = (end - from + stride - 1) / stride;
  if (end <= from) return;
  const int lane = threadIdx.x & 63, h = lane >> 4;
  const int32_t* table = a.c.table + r.i * a.c.table_row;
  const int per = a.c.shift - 5;  // log2 of a page's blocks
  // Lane l has the page of the l-th of 64 steps, none (-1) where it is not there.
  auto block_of = [&](int n) { return blocks.block(from + stride * min(n, steps - 1)); };
  int ids = 0;
  // (Blocks past the last, and in pages that are not there, are loaded from places that are.)
  auto load = [&](Raw<D>& raw, int n) {
    if ((n & 63) == 0) {
      const int page = table[block_of(n + lane) >> per];
      ids = n + lane < steps && (unsigned)page < (unsigned)a.c.pages ? page : -1;
    }
    const int page = __builtin_amdgcn_readlane(ids, n & 63);
    raw.load(a.c.data + a.c.head<D>(max(page, 0), kvh), a.c.shift, (block_of(n) & ((1 << per) - 1)) << 5, lane);
    return page >= 0;
  };
  auto step = [&](Raw<D>& raw, int n) {
    const int j0 = block_of(n) << 5;
    const bool hide = j0 + 32 > first.hi || (j0 < last.lo && j0 + 32 > a.sinks);
    uint32_t seen[QT] = {}, any = 255;
    if (hide) {
      any = seen8(j0 + 8 * h, Seen(first.lo, last.hi), a.sinks);
#pragma unroll
      for (int i = 0; i < QT; ++i) seen[i] = seen8(j0 + 8 * h, Seen(lo[i], hi[i]), a.sinks);
    }
    attend<CAREFUL>(acc, raw, a.scale2, hide, seen, any);
  };
  // The next step's codes are in flight while one is worked on. (Two steps ahead, with
  // registers moved from step to step, 64 tokens over their caches took 222 us, one
  // ahead 218, without the moves 213.)
  Raw<D> raw[2];
  bool there[2];
  there[0] = load(raw[0], 0);
  for (int n = 0; n < steps; n += 2) {
    there[1] = load(raw[1], n + 1);
    if (there[0]) step(raw[0], n);
    if (n + 1 >= steps) break;
    there[0] = load(raw[0], n + 2);
    if (there[1]) step(raw[1], n + 1);
  }
}

// Sums of waves and pieces, 64 at most, are joined as shares of 2^-kJoined and less, so
// that finite ones add up to a finite one.
constexpr float kJoined = 7.f;

// Sums of a piece of a tile's keys: the rows' references and sums, and their
// output values.
struct Partials {
  float2* ml;  // [piece][row], null: not split
  float* o;    // [piece][row][D]
  int64_t rows;
  int splits, piece;  // most pieces of a tile, and the blocks of one, more where a tile has more
  __device__ __forceinline__ int size(int blocks) const { return max(piece, (blocks + splits - 1) / splits); }
  // This workgroup's piece of a query's head.
  __device__ __forceinline__ int64_t at(const AttendArgs& a, int query, int head) const {
    return rows * blockIdx.y + (int64_t)query * a.c.kv_heads * a.group + head;
  }
};

// Few rows: a workgroup takes 16 QT of them; its waves every WAVES-th block of keys,
// whose sums they add in LDS. Where a tile has more blocks than a piece, each piece
// is a workgroup, and a second kernel joins their sums.
//
// Bound by memory over long caches: 64 tokens over 1.08 GB of 4-bit keys and values 213
// us (5.1 TB/s; a copy reaches 4.9 to 5.2), one over 131072 keys 27 us (5.3 TB/s) and
// its join 4 to 5; by latency below. With one step in flight, a wait for each
// page's number and registers copied between the two files it was 408. The split
// by pieces and not by shares of each request's keys gave 293 -> 227.
template <typename T, int D, int QT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, QT == 1 ? 3 : 2) void cache4_attention_kernel(AttendArgs a, Partials part) {
  constexpr int C = D / 16, W = D / 32;
  typedef typename Mma16<T>::frag frag;
  __shared__ __attribute__((aligned(16))) float sums[WAVES][16][D];  // of 16 rows at a time
  __shared__ float2 ml[WAVES][16];
  __shared__ __attribute__((aligned(16))) uint8_t queries[Rows16<T, D, QT>::IMAGE ? 16 * QT * 2 * D : 16];
  const int kvh = blockIdx.x % a.c.kv_heads, tile_no = blockIdx.x / a.c.kv_heads, split = blockIdx.y;
  const Request r(a, tile_no, 16 * QT);
  if (r.i < 0) return;
  const int rows = r.queries * a.group, row0 = (tile_no - r.tile) * 16 * QT;
  if ((unsigned)row0 >= (unsigned)rows) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 4;
  auto window = [&](int row) { return Seen(a, r.behind + a.query(row), r.keys); };
  const Seen first = window(row0), last = window(min(row0 + 16 * QT, rows) - 1);
  const Blocks blocks(a, first, last);
  const int size = part.size(blocks.n), block0 = size * split, block1 = min(blocks.n, block0 + size);
  if (block0 >= blocks.n && split) return;
  const bool whole = blocks.n <= size;  // the tile's only piece
  const int head_of = kvh * a.group;  // query head of row 0 of a query
  auto query_at = [&](int row, int query) {
    return (const T*)a.b.q + (int64_t)(r.q0 + query) * a.b.q_row + (int64_t)(head_of + row - query * a.group) * a.b.q_head;
  };
  Rows16<T, D, QT> acc;
  int lo[QT], hi[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int row = min(row0 + 16 * i + (lane & 15), rows - 1), query = a.query(row);
    const Seen s(a, r.behind + query, r.keys);
    lo[i] = s.lo;
    hi[i] = s.hi;
    if constexpr (!Rows16<T, D, QT>::IMAGE) {
#pragma unroll
      for (int w = 0; w < W; ++w) acc.held[w] = *(const frag*)(query_at(row, query) + h * (D / 4) + 8 * w);
    }
  }
  if constexpr (Rows16<T, D, QT>::IMAGE) {
    for (int at = threadIdx.x; at < 16 * QT * (D / 8); at += 64 * WAVES) {
      const int in = at / (D / 8), chunk = at % (D / 8), row = min(row0 + in, rows - 1);
      *(u32x4*)(queries + in * 2 * D + 16 * (chunk ^ (in & (D / 8 - 1)))) =
          *(const u32x4*)(query_at(row, a.query(row)) + 8 * chunk);
    }
    acc.image = queries;
    __syncthreads();
  }
  // (without pages there are no keys)
  const int from = block0 + wave, end = a.c.pages ? block1 : 0;
  attend_blocks<false>(a, acc, r, blocks, first, last, lo, hi, kvh, from, WAVES, end);
  if (acc.spoilt(lane)) attend_blocks<true>(a, acc, r, blocks, first, last, lo, hi, kvh, from, WAVES, end);
  // The waves' sums, 16 rows at a time.
  constexpr int THREADS = 64 * WAVES, PER = 16 * D / THREADS;  // columns of a thread
  static_assert(PER >= 4 && D % PER == 0, "whole vectors of one row");
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    acc.l[i] += __shfl_xor(acc.l[i], 16, 64);
    acc.l[i] += __shfl_xor(acc.l[i], 32, 64);
    if (i) __syncthreads();
    if (h == 0) ml[wave][lane & 15] = make_float2(acc.m[i], acc.l[i]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int t = 0; t < C; t += 4)
        *(float4v*)&sums[wave][lane & 15][(C * (4 * h + e) + t) ^ (4 * (lane & 7))] =
            float4v{acc.o[i][t][e], acc.o[i][t + 1][e], acc.o[i][t + 2][e], acc.o[i][t + 3][e]};
    __syncthreads();
    const int row = threadIdx.x * PER / D, c0 = threadIdx.x * PER % D, at = row0 + 16 * i + row;
    if (at >= rows) continue;
    float m = -INFINITY, l = 0.f, v[PER] = {};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, ml[w][row].x);
    m += kJoined;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float2 s = ml[w][row];
      if (s.x == -INFINITY && s.y == 0.f) continue;  // saw nothing
      const float f = s.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(s.x - m);
      l = fmaf(f, s.y, l);
#pragma unroll
      for (int c = 0; c < PER; c += 4) {
        const float4v o = *(const float4v*)&sums[w][row][(c0 + c) ^ (4 * (row & 7))];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[c + e] = fmaf(f, o[e], v[c + e]);
      }
    }
    const int query = a.query(at), head = head_of + at - query * a.group;
    if (!whole) {
      const int64_t to = part.at(a, r.q0 + query, head);
      if (c0 == 0) part.ml[to] = make_float2(m, l);
#pragma unroll
      for (int c = 0; c < PER; c += 4)
        *(float4v*)(part.o + to * D + c0 + c) = float4v{v[c], v[c + 1], v[c + 2], v[c + 3]};
    } else {
      typedef T vec __attribute__((ext_vector_type(4)));
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      T* out = (T*)a.b.out + (int64_t)(r.q0 + query) * a.b.out_row + (int64_t)head * a.b.out_head + c0;
#pragma unroll
      for (int c = 0; c < PER; c += 4)
        *(vec*)(out + c) = vec{(T)(v[c] * inv), (T)(v[c + 1] * inv), (T)(v[c + 2] * inv), (T)(v[c + 3] * inv)};
    }
  }
}

// Joins the pieces, at most 64, of tiles of `of` rows: WAVES waves of a workgroup take a
// row. Lane l of wave w adds columns 4 (l % (D / 4)) .. of every G WAVES-th piece from
// l / (D / 4) + G w on; the sums are added in order.
template <typename T, int D, int WAVES>
__global__ __launch_bounds__(256) void cache4_join_kernel(AttendArgs a, Partials part, int of, int items) {
  constexpr int C = D / 4, G = 64 / C;
  __shared__ float4v sums[WAVES][C];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int item = blockIdx.x * (4 / WAVES) + wave / WAVES, w = wave % WAVES;
  if (item >= items) return;  // (one row a workgroup, or a wave each: no barrier is left behind)
  const int kvh = item % a.c.kv_heads, tile_no = item / a.c.kv_heads;
  const Request r(a, tile_no, 1);
  if (r.i < 0) return;
  const int row = tile_no - r.tile;
  if ((unsigned)row >= (unsigned)(r.queries * a.group)) return;
  const int row0 = row / of * of;
  const Blocks blocks(a, Seen(a, r.behind + a.query(row0), r.keys),
                      Seen(a, r.behind + a.query(min(row0 + of, r.queries * a.group) - 1), r.keys));
  const int size = part.size(blocks.n), pieces = (blocks.n + size - 1) / size;
  if (pieces <= 1) return;  // the row is written
  const int i = a.query(row), head = kvh * a.group + (row - i * a.group);
  const int64_t at = (int64_t)(r.q0 + i) * a.c.kv_heads * a.group + head;
  // every wave: lane z's piece
  const float2 ml = lane < pieces ? part.ml[part.rows * lane + at] : make_float2(-INFINITY, 0.f);
  const int c = lane % C, g = lane / C;
  constexpr int BATCH = 8;  // pieces whose values are on their way together
  float4v o[BATCH];
  auto load = [&](int z0) {
#pragma unroll
    for (int k = 0; k < BATCH; ++k)
      o[k] = *(const float4v*)(part.o + (part.rows * min(z0 + k * G * WAVES + g, pieces - 1) + at) * D + 4 * c);
  };
  load(G * w);
  float m = ml.x;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
  m += kJoined;
  const bool empty = ml.x == -INFINITY && ml.y == 0.f;  // saw nothing
  const float f = empty ? 0.f : ml.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - m);
  float l = empty ? 0.f : f * ml.y;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) l += __shfl_xor(l, x, 64);
  const float weight = empty ? -1.f : f;
  float4v v = {0.f, 0.f, 0.f, 0.f};
  for (int z0 = G * w; z0 < pieces; z0 += BATCH * G * WAVES) {
    if (z0 > G * w) load(z0);
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int z = z0 + k * G * WAVES + g;
      const float of_z = __shfl(weight, z & 63, 64), by = z < pieces ? of_z : -1.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = by == -1.f ? v[e] : fmaf(by, o[k][e], v[e]);
    }
  }
#pragma unroll
  for (int x = C; x < 64; x *= 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += __shfl_xor(v[e], x, 64);
  if constexpr (WAVES > 1) {
    if (g == 0) sums[w][c] = v;
    __syncthreads();
    if (w) return;
    v = sums[0][c];
#pragma unroll
    for (int k = 1; k < WAVES; ++k) v += sums[k][c];
  }
  if (g) return;
  typedef T vec __attribute__((ext_vector_type(4)));
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  T* out = (T*)a.b.out + (int64_t)(r.q0 + i) * a.b.out_row + (int64_t)head * a.b.out_head;
  *(vec*)(out + 4 * c) = vec{(T)(v[0] * inv), (T)(v[1] * inv), (T)(v[2] * inv), (T)(v[3] * inv)};
}

// 16 rows from `begin` on over the blocks [block0, block1) of a tile's list, by one wave;
// those whose bit of `mask` is set are written. `low`: what spoilt rows begin with.
template <typename T, int D>
__device__ __forceinline__ void careful_rows(const AttendArgs& a, const Partials& part, const Request& r,
                                             const Blocks& blocks, const Seen& first, const Seen& last, int kvh,
                                             int begin, int rows, uint32_t mask, int block0, int block1, bool whole,
                                             float low) {
  constexpr int C = D / 16, W = D / 32;
  typedef typename Mma16<T>::frag frag;
  const int lane = threadIdx.x & 63, h = lane >> 4;
  const int row = min(begin + (lane & 15), rows - 1), query = a.query(row), head = kvh * a.group + row - query * a.group;
  const Seen mine(a, r.behind + query, r.keys);
  const int lo[1] = {mine.lo}, hi[1] = {mine.hi};
  Rows16<T, D, 1> acc;
  const T* q = (const T*)a.b.q + (int64_t)(r.q0 + query) * a.b.q_row + (int64_t)head * a.b.q_head + h * (D / 4);
#pragma unroll
  for (int w = 0; w < W; ++w) acc.held[w] = *(const frag*)(q + 8 * w);
  acc.low[0] = low;
  while (true) {
    attend_blocks<true>(a, acc, r, blocks, first, last, lo, hi, kvh, block0, 1, a.c.pages ? block1 : 0);
    if (acc.HALF || low > 0.f || !acc.spoilt(lane)) break;
    low = 42.f;
  }
  acc.l[0] += __shfl_xor(acc.l[0], 16, 64);
  acc.l[0] += __shfl_xor(acc.l[0], 32, 64);
  if (begin + (lane & 15) >= rows || !(mask >> (lane & 15) & 1)) return;
  const float inv = !whole ? 1.f : acc.l[0] == 0.f ? 0.f : 1.0f / acc.l[0];
  T* out = (T*)a.b.out + (int64_t)(r.q0 + query) * a.b.out_row + (int64_t)head * a.b.out_head;
  const int64_t to = part.at(a, r.q0 + query, head);
  if (!whole && h == 0) part.ml[to] = make_float2(acc.m[0], acc.l[0]);
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int t = 0; t < C; ++t) {
      const int column = C * (4 * h + e) + t;
      if (whole) out[column] = (T)(acc.o[0][t][e] * inv);
      else part.o[to * D + column] = acc.o[0][t][e];
    }
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup of 4 waves takes 128, and 64 keys a round for all of
// them, as window attention's tiles do: scores one block ahead and the product
// with V one behind, on v_mfma_f32_32x32x16. Each wave decodes 16 keys of K and of
// V of a round, among its products, into the images of the round behind it; their
// codes are loaded a round before that.
//
// Bound by no unit alone: MFMAs take 45 % of the cycles, vector instructions 44, LDS 39,
// and two waves a SIMD (its registers and images leave no third) do not cover one another,
// which wait for a third of their cycles to issue. 2048 queries of 32 heads of 128
// behind 16000 keys (8 KV heads) and three small requests, 575 GFLOP, take 534 to 574 us by
// the card, 1.0 PFLOP/s. Waves that decode all keys for
// 64 rows of their own, without LDS, took 775: decoding is then half of their
// instructions.
// ---------------------------------------------------------------------------

// What a wave decodes: 16 tokens' codes. K: lane l has quarter l % 4 of key l / 4; V:
// piece l % 16 of 4 tokens from 4 (l / 16) on.
template <typename T, int D>
struct Sixteen {
  static constexpr int W = D / 32, ITEMS = W + 4;
  typedef uint32_t vec __attribute__((ext_vector_type(W)));
  typedef Mma16<T> M;
  vec k, v;
  uint32_t k_scale, v_scales;
  // Tokens t .. t + 15 of a page whose KV head begins at `head`.
  __device__ __forceinline__ void load_k(const uint8_t* head, int t, int shift, int lane) {
    typedef Cache4Head<D> Head;
    const int key = t + (lane >> 2), quarter = lane & 3;
    k = *(const vec*)(head + Head::k_codes(key) + quarter * (D / 8));
    k_scale = head[Head::scale(shift, false, key, quarter * (D / 32) / 4)];
  }
  __device__ __forceinline__ void load_v(const uint8_t* head, int t, int shift, int lane) {
    typedef Cache4Head<D> Head;
    const int first = t + 4 * (lane >> 4), piece = lane & 15;
    v = *(const vec*)(head + Head::v_codes(shift, first, piece));
    v_scales = *(const uint32_t*)(head + Head::scale(shift, true, first, piece * (D / 32) / 16));
  }
  // Zeros for the values whose bit of `keep` is not set.
  __device__ __forceinline__ void drop(uint32_t keep) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (keep >> e & 1) continue;
      v_scales &= ~(255u << (8 * e));
      if constexpr (D == 128) v[e] = 0;
      else v[e >> 1] &= e & 1 ? 0xffffu : 0xffff0000u;
    }
  }
  // Item i of ITEMS into images of which the tokens are rows `row0` ...
  __device__ __forceinline__ void write(int i, uint8_t* k_image, uint8_t* v_image, int row0, int lane) const {
    if (i < W) {
      const float power = __uint_as_float(k_scale << 23);
      const uint32_t c = k[i];
      const u32x4 f = {M::template decode<0>(c, power), M::template decode<1>(c, power), M::template decode<2>(c, power),
                       M::template decode<3>(c, power)};
      const int row = row0 + (lane >> 2), chunk = W * (lane & 3) + i;
      *(u32x4*)(k_image + row * 2 * D + 16 * (chunk ^ k_swizzle<D>(row))) = f;
      return;
    }
    const int e = i - W, row = row0 + 4 * (lane >> 4) + e, piece = lane & 15;
    const int s = 23 - 8 * e;
    const float power = __uint_as_float(s >= 0 ? v_scales << s : v_scales >> -s);
    if constexpr (D == 128) {
      const uint32_t c = v[e];
      const u32x4 f = {M::template decode<0>(c, power), M::template decode<1>(c, power), M::template decode<2>(c, power),
                       M::template decode<3>(c, power)};
      *(u32x4*)(v_image + row * 2 * D + 16 * (piece ^ v_swizzle<D>(row))) = f;
    } else {
      const uint32_t c = e & 1 ? v[e >> 1] >> 16 : v[e >> 1];
      const u32x2 f = {M::template decode<0>(c, power), M::template decode<1>(c, power)};
      *(u32x2*)(v_image + row * 2 * D + 16 * ((piece >> 1) ^ v_swizzle<D>(row)) + 8 * (piece & 1)) = f;
    }
  }
};

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void cache4_tile_kernel(AttendArgs a, Partials part) {
  constexpr int IMG = 2 * kKeys * D, ROWS = 128;
  __shared__ __attribute__((aligned(16))) uint8_t lds[2][2][2 * IMG];  // [K, V][round & 1]
  __shared__ __attribute__((aligned(16))) uint8_t extra[IMG];          // K of the first block
  const int kvh = blockIdx.x % a.c.kv_heads, tile_no = blockIdx.x / a.c.kv_heads;
  const Request r(a, tile_no, ROWS);
  if (r.i < 0) return;
  const int rows = r.queries * a.group, row0 = (tile_no - r.tile) * ROWS;
  if ((unsigned)row0 >= (unsigned)rows) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hl = lane >> 5;
  auto window = [&](int row) { return Seen(a, r.behind + a.query(row), r.keys); };
  const Seen all_first = window(row0), all_last = window(min(row0 + ROWS, rows) - 1);
  const Blocks blocks(a, all_first, all_last);
  const int size = part.size(blocks.n), block0 = size * blockIdx.y, block1 = min(blocks.n, block0 + size);
  if (block0 >= blocks.n && blockIdx.y) return;
  const bool whole = blocks.n <= size;               // the tile's only piece
  const int count = a.c.pages ? block1 - block0 : 0;  // (without pages there are no keys)
  // In slots of the piece's list of blocks a row sees t < hi with t >= lo or t < sinks. (A
  // round may have a block behind the piece, which the next one has.)
  const int before = 32 * block0, sinks = a.sinks - before;
  auto listed = [&](int row) {
    const Seen s = window(row);
    return Seen(s.lo - 32 * blocks.skip - before, min(s.hi - 32 * blocks.skip - before, 32 * count));
  };
  const int w0 = row0 + 32 * wave, w1 = min(w0 + 31, rows - 1), row = min(w0 + (lane & 31), rows - 1);
  const Seen mine = listed(row), first = listed(min(w0, rows - 1)), last = listed(w1);
  const int rounds = (count + 1) >> 1, head_of = kvh * a.group;
  auto query_at = [&](int at) {
    const int i = a.query(at);
    return (const T*)a.b.q + (int64_t)(r.q0 + i) * a.b.q_row + (int64_t)(head_of + at - i * a.group) * a.b.q_head;
  };
  auto output = [&](int at) {
    const int i = a.query(at);
    return (T*)a.b.out + (int64_t)(r.q0 + i) * a.b.out_row + (int64_t)(head_of + at - i * a.group) * a.b.out_head;
  };
  const int32_t* table = a.c.table + r.i * a.c.table_row;
  const int per = a.c.shift - 5;  // log2 of a page's blocks
  auto block_of = [&](int b) { return blocks.block(block0 + max(0, min(b, count - 1))); };
  auto page_of = [&](int b) { return table[block_of(b) >> per]; };
  // Pages that are not there are the slow path's.
  bool missing = false;
  if (count) {
    for (int b = lane << per; b < count + (1 << per); b += 64 << per)
      if ((unsigned)page_of(b) >= (unsigned)a.c.pages) missing = true;
    // the sinks' last and the window's first, which those steps may pass over
    if ((unsigned)page_of(blocks.sinks - 1 - block0) >= (unsigned)a.c.pages) missing = true;
    if ((unsigned)page_of(blocks.sinks - block0) >= (unsigned)a.c.pages) missing = true;
  }
  missing = __builtin_amdgcn_ballot_w64(missing) != 0;
  uint8_t* const rows_image = lds[wave >> 1][1] + (wave & 1) * IMG;
  Rows<T, D> acc;
  acc.clear();
  if (!missing) {
    // The wave decodes tokens 16 (wave % 2) .. of K's block 2 at + 1 + wave / 2 and V's
    // 2 at - 1 + wave / 2 for round `at`.
    const int second = wave >> 1, sixteen = 16 * (wave & 1);
    Sixteen<T, D> codes;
    auto head_at = [&](int page) { return a.c.data + a.c.head<D>(page, kvh); };
    auto token = [&](int b) { return ((block_of(b) & ((1 << per) - 1)) << 5) + sixteen; };
    // Values that no row sees are zeros.
    auto seen = [&](int b) {
      const bool listed = b >= 0 && b < count;
      const int key = (block_of(b) << 5) + sixteen;
      if (listed && (key >= all_first.lo || key + 16 <= a.sinks) && key + 16 <= all_last.hi) return;
      asm volatile("");
      uint32_t keep = 0;
      if (listed)
        keep = seen8(key + 4 * (lane >> 4), Seen(all_first.lo, all_last.hi), a.sinks);
      codes.drop(keep);
    };
    int pages[2];  // of the V block that is loaded next, and of the K block
    int coming;    // of the K block behind it, on its way
    if (rounds) {
      // K of the first block, by waves 0 and 1
      const int p0 = __builtin_amdgcn_readfirstlane(page_of(0));
      codes.load_k(head_at(p0), token(0), a.c.shift, lane);
      if (!second) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) codes.write(i, extra, extra, sixteen, lane);
      }
      image_rows<D>(lane, [&](int i, int r, int chunk) {
        *(u32x4*)(rows_image + 1024 * i + 16 * lane) =
            *(const u32x4*)(query_at(min(w0 + r, rows - 1)) + 8 * (chunk ^ k_swizzle<D>(r)));
      });
      pages[0] = __builtin_amdgcn_readfirstlane(page_of(second - 1));
      pages[1] = __builtin_amdgcn_readfirstlane(page_of(second + 1));
      coming = page_of(second + 3);
      codes.load_k(head_at(pages[1]), token(second + 1), a.c.shift, lane);
      codes.load_v(head_at(pages[0]), token(second - 1), a.c.shift, lane);
      seen(second - 1);
#pragma unroll
      for (int i = 0; i < Sixteen<T, D>::ITEMS; ++i)
        codes.write(i, lds[0][0] + second * IMG, lds[1][0] + second * IMG, sixteen, lane);
    }
    auto landed = [&] {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      meet();
    };
    // Codes of round `at`, whose V's pages are those of K's before.
    auto load = [&](int at) {
      pages[0] = pages[1];
      pages[1] = __builtin_amdgcn_readfirstlane(coming);
      coming = page_of(2 * at + 3 + second);
      codes.load_k(head_at(pages[1]), token(2 * at + 1 + second), a.c.shift, lane);
      codes.load_v(head_at(pages[0]), token(2 * at - 1 + second), a.c.shift, lane);
    };
    float16v s;
    auto hidden = [&](int t0) {
      if (t0 + 32 > first.hi || (t0 < last.lo && t0 + 32 > sinks)) {
        asm volatile("");
        hide(s, t0, hl, mine.lo, mine.hi, sinks);
      }
    };
    typename Mma<T>::frag p[2] = {};
    if (rounds) {
      load(1);
      landed();
      acc.load(rows_image, lane);
      s = acc.scores(extra, lane);
      hidden(0);
    }
    for (int at = 0; at < rounds; ++at) {
      landed();  // the round's images, and every wave has left the others
      const int odd = at & 1;
      constexpr int C = D / 16, CALLS = 2 * C, ITEMS = Sixteen<T, D>::ITEMS;
      static_assert(ITEMS < CALLS, "a call for each item, and one for the loads");
      seen(2 * at + 1 + second);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        acc.step(s, p, lds[1][odd] + k * IMG, lds[0][odd] + k * IMG, lane, a.scale2, [&](int c) {
          const int call = C * k + c;
          if (call < ITEMS) codes.write(call, lds[0][1 - odd] + second * IMG, lds[1][1 - odd] + second * IMG, sixteen, lane);
          else if (call == ITEMS) load(at + 2);
        });
        hidden(64 * at + 32 + 32 * k);
      }
    }
    if (rounds && 2 * rounds == count) {
      landed();
      acc.values(lds[1][rounds & 1], lane, p);
    }
    acc.l += __shfl_xor(acc.l, 32, 64);
  }
  // Rows whose sums are not finite, which a value that they do not see may be
  // the cause of, and rows over pages that are not there are taken again.
  const uint64_t bad = missing ? ~0ull : __builtin_amdgcn_ballot_w64(acc.spoilt());
  const uint32_t again = (uint32_t)(bad | bad >> 32);
  if (whole) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    meet();
    acc.store((T*)(rows_image + (lane & 31) * 2 * D), lane & 31, hl);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    image_rows<D>(lane, [&](int i, int r, int chunk) {
      const u32x4 v = *(const u32x4*)(rows_image + r * 2 * D + 16 * (chunk ^ k_swizzle<D>(r)));
      if (w0 + r < rows && !(again >> r & 1)) *(u32x4*)(output(w0 + r) + 8 * chunk) = v;
    });
  } else if (w0 + (lane & 31) < rows && !(again >> (lane & 31) & 1)) {
    const int i = a.query(row);
    const int64_t to = part.at(a, r.q0 + i, head_of + row - i * a.group);
    if (hl == 0) part.ml[to] = make_float2(acc.m, acc.l);
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *(float4v*)(part.o + to * D + 32 * db + 8 * j + 4 * hl) =
            float4v{acc.o[db][4 * j], acc.o[db][4 * j + 1], acc.o[db][4 * j + 2], acc.o[db][4 * j + 3]};
  }
  if (again) {
    asm volatile("");
    for (int i = 0; i < 2; ++i) {
      const uint32_t mask = again >> (16 * i) & 0xffff;
      const int begin = w0 + 16 * i;
      if (mask && begin < rows)
        careful_rows<T, D>(a, part, r, blocks, all_first, all_last, kvh, begin, rows, mask, block0, block1, whole,
                           missing ? 0.f : 42.f);
    }
  }
}

// Rows of a tile and how the keys are split, by a batch's sizes alone (us, 32 heads of
// 128, 8 KV heads; tiles of 16 : 32 : 128 rows).
//  Requests of up to 32 rows: 16 (32 x 8 queries, 5000 keys 60 : 78 : 107, 8 over 60000 keys
//  33 : 41 : 45; one of 4, 5000 keys 13.5 : 14.3 : 21).
//  From 256 rows on, with 512 tiles of 128 or, all together, 32768 blocks of keys: 128 (16
//  x 100 queries of 100 keys 26 : 25 : 16, 2048 of 2048 88 : 75 : 65, 128 over 60000 keys 260 :
//  187 : 149).
//  Between: 32 (32 x 32, 5000 keys 172 : 136 : 190; 512 of 512 15 : 12.5 : 18; 64 over 5000
//  keys 27 : 24 : 28; 128 over 5000 34 : 31 : 35; 512 over 5000 83 : 66 : 68).
// A split costs a second launch and is taken from 48 blocks on, 72 where there are 128
// tiles (one token: 5000 keys 19.6 whole, 12.4 in pieces of 16 blocks, 2000 keys 16.0 and
// 12.4, 1400 12.3 and 12.7; 200 queries, 2000 keys 23 and 33), into pieces that fill
// the chip 16 times over for single tokens, whose requests' lengths differ (64 tokens over
// their caches: 768 pieces 263, 1536 252, 2048 231, 4096 219 to 227, 8192 235), twice
// for more rows, whose sums are written and read again (512 over 5000 keys: 512 pieces
// 66, 1024 79, 4096 107), of 64 blocks at least where there is work for 1024 such
// (32 x 4 queries over 5000 keys in pieces of 16 blocks 80, of 39 63).
struct Plan {
  int rows, splits, piece;  // rows of a tile; most pieces of a tile, and the blocks of 32 keys of one
};
Plan plan_of(const nemo_attention_config& c, int count, int64_t q_rows, int64_t max_kv) {
  if (count == 0 || q_rows == 0) return {16, 1, 1};
  const int64_t rows = q_rows * (c.q_heads / c.kv_heads);
  auto tiles_of = [&](int n) { return std::max<int64_t>(rows / n, count) * c.kv_heads; };
  int64_t keys = max_kv;
  if (c.left >= 0 && c.right >= 0) keys = std::min(keys, (int64_t)c.left + c.right + 1 + c.sinks);
  const int64_t blocks = std::min<int64_t>(keys, 1 << 30) / 32 + 1;
  int tile = rows / count <= 32 ? 16 : 32;
  if (rows / count >= 256 && (tiles_of(128) >= 512 || blocks * tiles_of(128) >= 512 * 64)) tile = 128;
  const int64_t work = blocks * tiles_of(tile);
  if (blocks <= (tiles_of(tile) < 128 ? 48 : 72)) return {tile, 1, (int)blocks};
  const int64_t piece = std::max<int64_t>({16, std::min<int64_t>(64, work / 1024), work / (tile == 16 ? 4096 : 512) + 1,
                                           (blocks + 63) / 64});
  return {tile, (int)((blocks + piece - 1) / piece), (int)piece};
}

}  // namespace

size_t cache4_workspace(const nemo_attention_config& c, int count, int64_t q_rows, int64_t max_kv) {
  const int splits = plan_of(c, count, q_rows, max_kv).splits;
  return splits == 1 ? 0 : (size_t)splits * q_rows * c.q_heads * (c.head_dim * 4 + 8);
}

hipError_t launch_cache4_attention(const nemo_cache4_config& cache, const nemo_attention_config& c,
                                   const nemo_cache4_pages& p, const nemo_cache4_queries& b, hipStream_t stream) {
  if (p.count == 0 || b.q_rows == 0) return hipSuccess;
  AttendArgs a{b, Cache4(cache, p), c.q_heads / c.kv_heads, 0, 0, 0, 0.f, 0, 0};
  while (1 << a.shift < a.group) ++a.shift;
  a.magic = (uint32_t)((((uint64_t)1 << a.shift) - a.group) * ((uint64_t)1 << 32) / a.group + 1);
  auto bound = [](int v) { return v < 0 ? kUnbounded : std::min(v, kUnbounded); };
  a.left = bound(c.left);
  a.right = bound(c.right);
  a.sinks = std::min(c.sinks, kUnbounded);
  a.scale2 = (c.scale > 0.f ? c.scale : 1.0f / sqrtf((float)c.head_dim)) * 1.4426950408889634f;
  const Plan plan = plan_of(c, p.count, b.q_rows, b.max_kv);
  const int splits = b.workspace ? plan.splits : 1;
  const int64_t rows = b.q_rows * c.q_heads;
  Partials part{nullptr, nullptr, rows, splits, plan.piece};
  if (splits > 1) {
    part.o = (float*)b.workspace;
    part.ml = (float2*)(part.o + splits * rows * c.head_dim);
  }
  auto tiles = [&](int r) { return (unsigned)(b.q_rows * a.group / r + p.count) * c.kv_heads; };
  auto launch = [&](auto type, auto d) {
    constexpr int D = decltype(d)::value;
    typedef decltype(type) T;
    const dim3 grid(tiles(plan.rows), splits);
    if (plan.rows == 16) cache4_attention_kernel<T, D, 1, 4><<<grid, 256, 0, stream>>>(a, part);
    else if (plan.rows == 32) cache4_attention_kernel<T, D, 2, 4><<<grid, 256, 0, stream>>>(a, part);
    else cache4_tile_kernel<T, D><<<grid, 256, 0, stream>>>(a, part);
    if (splits == 1) return;
    // a workgroup a row for few of them, else a wave
    const int items = (int)tiles(1);
    if (items <= 2048) cache4_join_kernel<T, D, 4><<<items, 256, 0, stream>>>(a, part, plan.rows, items);
    else cache4_join_kernel<T, D, 1><<<(items + 3) / 4, 256, 0, stream>>>(a, part, plan.rows, items);
  };
  auto typed = [&](auto type) {
    if (c.head_dim == 64) launch(type, std::integral_constant<int, 64>{});
    else launch(type, std::integral_constant<int, 128>{});
  };
  if (c.type == NEMO_TYPE_F16) typed(half_t{});
  else typed(bf16_t{});
  return hipGetLastError();
}

}  // namespace nemo
