// Attention with a sliding window and sinks for gfx950 (include/nemo.h
// nemo_window_attention): softmax(scale q.k) v over the keys j <= p + right
// that have j >= p - left or j < sinks.
//
// Rows are (query, head of the group) pairs of one request and KV head, query
// by query, so 32 rows fill an MFMA operand whatever the group and the number
// of queries. A tile of rows attends a list of N key slots: the sinks before
// its first window key, then the keys of its rows' windows together; no other
// key is read. Scores are taken transposed, S^T = K Q^T (32 keys x 32 rows per
// v_mfma_f32_32x32x16), so a lane holds one row, its softmax is per-lane
// arithmetic in fp32, and its score registers are the B operand of O^T = V^T
// P^T: the MFMA's k slots of a 16-key chunk are taken in the order that the
// score registers have. K and V go row-major into LDS by DMA; K fragments are
// 16-byte reads, V^T fragments transposed reads (ds_read_b64_tr_b16).
#include <algorithm>
#include <type_traits>

#include "nemo_operators.h"

namespace nemo {

namespace {

struct WindowArgs {
  nemo_attention_batch b;
  int kv_heads, group, left, right, sinks;
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
  __device__ __forceinline__ Seen(const WindowArgs& a, int p, int n) {
    hi = max(0, min(n, a.right >= kUnbounded ? n : p + a.right + 1));
    lo = a.left >= kUnbounded ? 0 : min(hi, max(0, p - a.left));
  }
};

// A request as it lies in the buffers, whatever the index arrays hold, and the
// number of its first tile. Tiles of ROWS (query, head of the group) rows are
// numbered through a batch without a table: request i's first number is
// floor(q_start[i] group / ROWS) + i, which leaves it at least as many numbers
// as it has tiles. The request of tile number t is the last whose first is not
// above t; none (i = -1) before the first request. A wave looks at 64 requests
// at a time, evenly over those that it may be, until they are 64 or fewer; a
// lane then has the request's whole entry at hand. (Of entries that do not
// ascend it may be one whose first tile is behind t.)
template <int ROWS>
struct Request {
  int i, tile, q0, queries, keys;
  int64_t kv0;
  __device__ __forceinline__ Request(const WindowArgs& a, int t) {
    const nemo_attention_batch& b = a.b;
    const int lane = threadIdx.x & 63;
    auto row = [&](int at) { return min(max(b.q_start[at], 0), (int)b.q_rows); };
    auto number = [&](int begin, int at) { return (int)((int64_t)begin * a.group / ROWS) + at; };
    int from = 0, left = b.count;
    while (left > 64) {
      const int step = (left + 63) >> 6, at = from + min(lane * step, left - 1);
      const int n = (int)__popcll(__builtin_amdgcn_ballot_w64(lane * step < left && number(row(at), at) <= t));
      from += max(n - 1, 0) * step;
      left = min(step, b.count - from);
    }
    const int at = min(from + lane, b.count - 1), begin = row(at), end = min(b.q_start[at + 1], (int)b.q_rows);
    const int64_t kv = min(max(b.kv_start[at], (int64_t)0), b.kv_rows);
    const int len = (int)min((int64_t)max(b.kv_len[at], 0), b.kv_rows - kv), first = number(begin, at);
    const int n = (int)__popcll(__builtin_amdgcn_ballot_w64(lane < left && first <= t));
    i = from + n - 1;
    if (!n) i = -1;
    const int of = max(n - 1, 0);
    tile = __builtin_amdgcn_readlane(first, of);
    q0 = __builtin_amdgcn_readlane(begin, of);
    queries = max(__builtin_amdgcn_readlane(end, of) - q0, 0);
    keys = __builtin_amdgcn_readlane(len, of);
    kv0 = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)kv, of) |
          (int64_t)__builtin_amdgcn_readlane((int)(kv >> 32), of) << 32;
  }
};

// One query head over keys [j0, j1), by a wave: its running maximum, sum and
// output columns lane, lane + 64.
template <typename T, int HD>
struct OneRow {
  float m = -INFINITY, l = 0.f, o[HD / 64] = {};
  __device__ __forceinline__ void keys(const T* q, const T* k, int64_t k_row, const T* v, int64_t v_row, int j0,
                                       int j1, float scale2) {
    typedef T vec __attribute__((ext_vector_type(8)));
    const int lane = threadIdx.x & 63;
    for (int jb = j0; jb < j1; jb += 64) {
      const int j = min(jb + lane, j1 - 1);
      float s = 0.f;
      for (int d = 0; d < HD; d += 8) {
        const vec a = *(const vec*)(q + d), b = *(const vec*)(k + j * k_row + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf((float)a[e], (float)b[e], s);
      }
      s = jb + lane < j1 ? s * scale2 : -INFINITY;
      float most = s;
      for (int x = 32; x > 0; x >>= 1) most = fmaxf(most, __shfl_xor(most, x, 64));
      const float mn = fmaxf(m, most), ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = exp2f(m - ref), p = jb + lane < j1 ? exp2f(s - ref) : 0.f;
      float sum = p;
      for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x, 64);
      l = l * alpha + sum;
      m = mn;
      for (int i = 0; i < HD / 64; ++i) o[i] *= alpha;
      for (int t0 = 0; t0 < min(64, j1 - jb); t0 += 8) {
        float r[8][HD / 64];
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
          for (int i = 0; i < HD / 64; ++i) r[t][i] = (float)v[min(jb + t0 + t, j1 - 1) * v_row + lane + 64 * i];
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const float pt = __shfl(p, t0 + t, 64);
#pragma unroll
          for (int i = 0; i < HD / 64; ++i) o[i] = jb + t0 + t < j1 ? fmaf(pt, r[t][i], o[i]) : o[i];
        }
      }
    }
  }
  __device__ __forceinline__ void store(T* out) const {
    for (int i = 0; i < HD / 64; ++i) out[(threadIdx.x & 63) + 64 * i] = (T)(l == 0.f ? 0.f : o[i] / l);
  }
};

// ---------------------------------------------------------------------------
// Fragments
// ---------------------------------------------------------------------------

typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef float float8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) short4v lds_short4v;

template <typename T>
struct Mma;
template <>
struct Mma<half_t> {
  typedef half8v frag;
  typedef half2v pair;
  static __device__ __forceinline__ float add(pair p, float sum) {
    return __builtin_amdgcn_fdot2(p, pair{(half_t)1.f, (half_t)1.f}, sum, false);
  }
  static __device__ __forceinline__ float16v mma(frag a, frag b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<bf16_t> {
  typedef bf16x8 frag;
  typedef bf16_t pair __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ float add(pair p, float sum) {
    return __builtin_amdgcn_fdot2_f32_bf16(p, pair{(bf16_t)1.f, (bf16_t)1.f}, sum, false);
  }
  static __device__ __forceinline__ float16v mma(frag a, frag b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

// LDS images of 32 keys, row-major, HD / 8 chunks of 16 bytes a row, chunk c of
// row r at c ^ swizzle: K's spreads the 32 rows that a fragment read touches
// over the banks, V's the four rows of 64 bytes of a transposed read.
constexpr int kKeys = 32;
template <int HD>
__device__ __forceinline__ int k_swizzle(int row) {
  return HD == 128 ? row & 15 : (row & 7) ^ ((row >> 3) & 1);
}
template <int HD>
__device__ __forceinline__ int v_swizzle(int row) {
  return HD == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1);
}

// Copies of 16 bytes a lane into LDS at `to` + 16 lane, from a buffer's range
// (zeros past its end) or an address. The compiler, which knows of the builtin for this that
// it writes LDS, waits for every copy in flight before each transposed read;
// written as here it has no register to be waited for, and the loops wait
// for their images themselves. (m0 is reserved: the compiler sets it where it
// uses it itself.)
__device__ __forceinline__ uint32_t lds_address(const uint8_t* to) { return (uint32_t)(uintptr_t)(lds_void*)to; }
__device__ __forceinline__ void copy_range(u32x4 range, uint32_t offset, const uint8_t* to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds_address(to)), "v"(offset), "s"(range)
               : "memory");
}
__device__ __forceinline__ void copy_address(const void* from, const uint8_t* to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(lds_address(to)), "v"(from)
               : "memory");
}
// A barrier that waits for none of the wave's work in flight; no access of
// memory is moved over it.
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Copies of ROWS key rows into an image by one wave, 1 KB an instruction:
// rows first .. first + ROWS of a 32-row image (or of two that follow each
// other). off: the lane's byte offsets from row 0 of the image, for rows that
// lie `stride` bytes apart.
template <int HD, int ROWS, bool VALUES>
struct Stager {
  static constexpr int kChunks = HD / 8, kPer = 64 / kChunks, kN = ROWS / kPer;
  uint32_t off[kN];
  int row;
  __device__ __forceinline__ Stager(int first, int64_t stride) {
    const int lane = threadIdx.x & 63;
    row = first + lane / kChunks;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int r = row + kPer * i;
      off[i] = (uint32_t)(r * stride) + 16 * ((lane % kChunks) ^ (VALUES ? v_swizzle<HD>(r) : k_swizzle<HD>(r)));
    }
  }
  // The image of the rows from `at` on, of which `valid` are copied and the
  // others zero.
  static __device__ __forceinline__ u32x4 range(const uint8_t* at, int64_t stride, int valid) {
    const int bytes = (int)stride * max(0, min(valid, kKeys));
    return u32x4{(uint32_t)(uintptr_t)at, (uint32_t)((uintptr_t)at >> 32) & 0xffffu,
                 (uint32_t)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
  }
  __device__ __forceinline__ void copy(u32x4 range, int i, const uint8_t* image) const {
    copy_range(range, off[i], image + 1024 * i);
  }
  __device__ __forceinline__ void copy(u32x4 range, const uint8_t* image) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) copy(range, i, image);
  }
};

// The key list of the rows of queries at p0 .. p1: slots t < sinks are keys t,
// slots from `pad`, a multiple of 32, on the keys from lo on, and those between
// are empty, so an image of 32 slots holds rows that follow each other. In
// list coordinates a row sees t < hi with t >= lo or t < sinks.
struct KeyList {
  int pad, lo, n, all_sinks;
  __device__ __forceinline__ KeyList(const WindowArgs& a, int p0, int p1, int keys) {
    const Seen first(a, p0, keys), last(a, p1, keys);
    all_sinks = a.sinks;
    lo = a.sinks < first.lo ? first.lo : 0;  // sinks that reach the window: keys from 0 on
    pad = lo ? (a.sinks + 31) & ~31 : 0;
    n = pad + last.hi - lo;
  }
  __device__ __forceinline__ int key(int t) const { return t < pad ? t : lo + t - pad; }
  // Rows that the image of the slots t0 .. t0 + 31 has.
  __device__ __forceinline__ int rows(int t0) const { return t0 < 0 ? 0 : (t0 < pad ? all_sinks : n) - t0; }
  __device__ __forceinline__ Seen window(const WindowArgs& a, int p, int keys) const {
    Seen s(a, p, keys);
    s.lo += pad - lo;
    s.hi += pad - lo;
    return s;
  }
};

// A wave's 32 rows: row l % 32 in lane l, whose half hl = l / 32 holds the
// output columns 32 db + 8 j + 4 hl + 0..3 in registers 4j.. of o[db], and the
// sum of its own keys' probabilities.
template <typename T, int HD>
struct Rows {
  static constexpr int DC = HD / 16, DB = HD / 32;
  typedef typename Mma<T>::frag frag;
  frag q[DC];
  float16v o[DB];
  float m, l;  // reference and sum of the probabilities

  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
  }
  __device__ __forceinline__ void load(const uint8_t* image, int lane) {
#pragma unroll
    for (int c = 0; c < DC; ++c) q[c] = key(image, lane, c);
  }
  __device__ __forceinline__ frag key(const uint8_t* image, int lane, int c) const {
    const int row = lane & 31;
    return *(const frag*)(image + row * 2 * HD + 16 * ((2 * c + (lane >> 5)) ^ k_swizzle<HD>(row)));
  }
  __device__ __forceinline__ float16v scores(const uint8_t* image, int lane) const {
    float16v s = {};
#pragma unroll
    for (int c = 0; c < DC; ++c) s = Mma<T>::mma(key(image, lane, c), q[c], s);
    return s;
  }
  // Probabilities 2^(s - m) are taken against a reference m that lay BELOW under
  // the row's largest score when it was last raised: it is raised when the sum
  // of a lane's 16 passes MOST (or is not a number, as for a row that has seen
  // nothing, whose m is -infinity), and they are taken again. So the common
  // block needs no maximum, no exchange between lanes and no rescaling, and one
  // wave vote. Numerator and denominator share the reference, so the result is
  // the softmax; the sum is that of the rounded probabilities.
  //
  // Half precision rounds what is below 2^-14 by up to 2^-25 whatever it is:
  // with a largest probability of 2^8 and more that is 2^-33 of it, and a long
  // cache of even scores that lie 17 under a sink's keeps its share of the
  // result (with a largest one of 1, e^-17 became 2^-24, 44 % more). Its MOST
  // is what no sum of finite ones reaches, so the raise comes when one
  // overflows: at 2^15, as for bf16, the headroom lost cost the 16 ragged
  // requests 0.6 us; now they take what they took without BELOW.
  static constexpr bool HALF = std::is_same<T, half_t>::value;
  static constexpr float BELOW = HALF ? 8.f : 0.f, MOST = HALF ? 0x1p20f : 0x1p15f;
  static __device__ __forceinline__ float sum(const frag (&p)[2]) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v = Mma<T>::add(typename Mma<T>::pair{p[i >> 2][2 * (i & 3)], p[i >> 2][2 * (i & 3) + 1]}, v);
    return v;
  }
  static __device__ __forceinline__ void exponentials(const float16v& s, float scale2, float m, frag (&p)[2]) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float8v e;
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(s[8 * c + i], scale2, -m));
      p[c] = __builtin_convertvector(e, frag);
    }
  }
  // Adds the sum of p, the probabilities of s, to the row's, after raising the
  // reference where it has to be.
  __device__ __forceinline__ void settle(const float16v& s, float scale2, frag (&p)[2]) {
    float add = sum(p);
    if (__builtin_amdgcn_ballot_w64(!(add <= MOST))) {
      asm volatile("");  // keeps the rare path a branch
      float top = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
      top *= scale2;
      const int high = !(add <= MOST), other = __shfl_xor(high, 32, 64);
      const bool raise = high | other;  // only the rows that ask: none depends on another
      const float raised = raise ? fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)) - BELOW) : m;
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - raised);
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
      m = raised;
      exponentials(s, scale2, m == -INFINITY ? 0.f : m, p);
      add = sum(p);
    }
    l += add;
  }
  // V^T fragment of 16 keys (chunk c) and 32 columns (block db): k slot 8 hl +
  // e is key 16 c + 8 (e / 4) + 4 hl + e % 4, that of score register 8 c + e. A
  // transposed read gives the 16 lanes of a group 4 keys of 16 columns; lane i
  // of it reads key i / 4's columns 4 (i % 4)...
  __device__ __forceinline__ frag value(const uint8_t* image, int lane, int c, int db) const {
    const int i = lane & 15, key = 4 * (lane >> 5) + (i >> 2);
    const int chunk = (4 * db + 2 * ((lane >> 4) & 1) + ((i >> 1) & 1)) ^ v_swizzle<HD>(key);
    const uint8_t* at = image + key * 2 * HD + 16 * chunk + 8 * (i & 1);
    short8v a;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const short4v v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4v*)(at + (16 * c + 8 * u) * 2 * HD));
#pragma unroll
      for (int e = 0; e < 4; ++e) a[4 * u + e] = v[e];
    }
    return __builtin_bit_cast(frag, a);
  }
  // O^T += V^T P^T
  __device__ __forceinline__ void values(const uint8_t* image, int lane, const frag (&p)[2]) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = Mma<T>::mma(value(image, lane, c, db), p[c], o[db]);
  }
  // One block of the pipelined loop: its probabilities from its scores s; in
  // the same stream of instructions the scores of the next block, from the
  // keys at k_image, and the product of the block before, whose
  // probabilities are p, with its values at v_image. Then s and p are those of
  // the next step. The matrix cores' work does not wait for the vector
  // units' that way, and a wave issues both in turn.
  // Copies (c), c < DC, are issued among the MFMAs too: a wave waits for the
  // memory pipe at each.
  template <typename Copies>
  __device__ __forceinline__ void step(float16v& s, frag (&p)[2], const uint8_t* v_image, const uint8_t* k_image,
                                       int lane, float scale2, Copies&& copies) {
    frag kf[DC], vf[DC], next[2];
    float16v n = {};
    auto exponentials = [&](int from, int to) {
#pragma unroll
      for (int r = from; r < to; r += 2) {
        float v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          v[i] = __builtin_amdgcn_exp2f(fmaf(s[r + i], scale2, -m));
          asm volatile("" : "+v"(v[i]));  // here, not together where they are used
        }
        next[r >> 3][r & 7] = (T)v[0];
        next[r >> 3][(r & 7) + 1] = (T)v[1];
      }
    };
    constexpr int AHEAD = DC / 2;  // fragments are read that many MFMAs before they are used
    auto fragment = [&](int c) {
      vf[c] = value(v_image, lane, c / DB, c % DB);  // first: the wait for the keys' is theirs too
      kf[c] = key(k_image, lane, c);
    };
#pragma unroll
    for (int c = 0; c < AHEAD; ++c) fragment(c);
    __builtin_amdgcn_sched_barrier(0);
    exponentials(0, 4);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      n = Mma<T>::mma(kf[c], q[c], n);
      exponentials(4 + 2 * (6 * c / DC), 4 + 2 * (6 * (c + 1) / DC));
      __builtin_amdgcn_sched_barrier(0);
      o[c % DB] = Mma<T>::mma(vf[c], p[c / DB], o[c % DB]);
      if (c + AHEAD < DC) fragment(c + AHEAD);
      copies(c);
      __builtin_amdgcn_sched_barrier(0);
    }
    settle(s, scale2, next);
    s = n;
    p[0] = next[0];
    p[1] = next[1];
  }
  // The lane's row into an image, at that image row.
  __device__ __forceinline__ void store(T* out, int row, int hl) const {
    typedef T vec __attribute__((ext_vector_type(4)));
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        vec v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(o[db][4 * j + e] * inv);
        *(vec*)(out + 8 * ((4 * db + j) ^ k_swizzle<HD>(row)) + 4 * hl) = v;
      }
  }
  // Whether a value of the lane's row is not finite.
  __device__ __forceinline__ bool spoilt() const {
    float z = l * 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) z = fmaf(o[db][r], 0.f, z);
    return z != 0.f;
  }
};

// Scores of hidden slots of the block at t0 become -infinity: bit c of `seen` is
// whether slot t0 + c is t < hi with t >= lo or t < sinks.
__device__ __forceinline__ void hide(float16v& s, int t0, int hl, int lo, int hi, int sinks) {
  auto below = [&](int t) {  // bits of the slots before t
    const int n = max(0, min(t - t0, 32));
    return n == 32 ? ~0u : (1u << n) - 1;
  };
  const uint32_t seen = (below(hi) & (~below(lo) | below(sinks))) >> (4 * hl);
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const uint32_t keep = (uint32_t)((int)(seen << (31 - 8 * (r >> 2) - (r & 3))) >> 31);
    s[r] = __uint_as_float((__float_as_uint(s[r]) & keep) | (0xff800000u & ~keep));
  }
}

// Addresses of one request and KV head.
template <typename T>
struct Heads {
  const T *q, *k, *v;
  T* out;
  int64_t q_row, q_head, out_row, out_head;
  int group;
  __device__ __forceinline__ Heads(const WindowArgs& a, int q0, int64_t kv0, int kvh)
      : q_row(a.b.q_row), q_head(a.b.q_head), out_row(a.b.out_row), out_head(a.b.out_head), group(a.group) {
    q = (const T*)a.b.q + q0 * q_row + (int64_t)kvh * group * q_head;
    k = (const T*)a.b.k + kv0 * a.b.k_row + kvh * a.b.k_head;
    v = (const T*)a.b.v + kv0 * a.b.v_row + kvh * a.b.v_head;
    out = (T*)a.b.out + q0 * out_row + (int64_t)kvh * group * out_head;
  }
  // Row `row`, of query i.
  __device__ __forceinline__ const T* query(int row, int i) const {
    return q + i * q_row + (row - i * group) * q_head;
  }
  __device__ __forceinline__ T* output(int row, int i) const {
    return out + i * out_row + (row - i * group) * out_head;
  }
};

// The rows of an image of 32, 16 bytes a lane: do(i, row, chunk) for row kPer i +
// lane / kChunks of the image and its chunk, i < HD / 16.
template <int HD, typename Do>
__device__ __forceinline__ void image_rows(int lane, Do&& each) {
  constexpr int kChunks = HD / 8, kPer = 64 / kChunks;
#pragma unroll
  for (int i = 0; i < kKeys / kPer; ++i) each(i, kPer * i + lane / kChunks, lane % kChunks);
}

// Whether, of the slots [t0, t1), one that not all rows of windows first ..
// last see has a value that is not finite: only then can their sums have met
// one that they do not see. By a wave.
template <typename T, int HD>
__device__ __forceinline__ bool hidden_spoil(const WindowArgs& a, const Heads<T>& h, const KeyList& list,
                                             const Seen& first, const Seen& last, int t0, int t1) {
  typedef T vec __attribute__((ext_vector_type(8)));
  constexpr int kChunks = HD / 8, kPer = 64 / kChunks;
  const int lane = threadIdx.x & 63;
  float z = 0.f;
  auto scan = [&](int from, int to) {
    for (int t = max(from, t0) + lane / kChunks; t < min(to, t1); t += kPer) {
      const vec v = *(const vec*)(h.v + list.key(t) * a.b.v_row + 8 * (lane % kChunks));
#pragma unroll
      for (int e = 0; e < 8; ++e) z = fmaf((float)v[e], 0.f, z);
    }
  };
  scan(list.pad ? list.pad : a.sinks, last.lo);
  scan(max(first.hi, list.pad), list.n);
  return __builtin_amdgcn_ballot_w64(z != 0.f) != 0;
}

// A row over the slots [t0, t1) that it sees, key by key.
template <typename T, int HD>
__device__ __forceinline__ OneRow<T, HD> one_row(const WindowArgs& a, const Heads<T>& h, const KeyList& list,
                                                 int queries, int keys, int row, int t0, int t1) {
  const int i = a.query(row);
  const Seen seen = list.window(a, keys - queries + i, keys);
  const int first = min(a.sinks, seen.hi);
  OneRow<T, HD> acc;
  acc.keys(h.query(row, i), h.k, a.b.k_row, h.v, a.b.v_row, t0, min(t1, first), a.scale2);
  const int from = max(max(t0, seen.lo), first), to = min(t1, seen.hi);
  if (from < to) acc.keys(h.query(row, i), h.k, a.b.k_row, h.v, a.b.v_row, list.key(from), list.key(to - 1) + 1, a.scale2);
  return acc;
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup of 4 waves takes 128 rows, 32 a wave, and stages 64
// keys a round for all of them. A block's scores are taken one block ahead and
// its product with V one behind, so the K rows of a round begin a block after
// the round's own, its V rows a block before.
//
// Where such tiles are too few for the chip, 8 waves take 64 rows: PARTS = 4
// pairs of waves attend a quarter of the keys each, 32 a round, and add up in
// LDS (requests of 512, 77, 1 and 300 tokens, 16 heads of 128 over up to 1040
// keys: 18.7 us; 24 with 128 rows or by window_few_kernel, 20 with two parts of
// two waves, of which a SIMD then has one).
//
// Bound by the steps' instructions and by power: 32768 tokens of 32 heads of
// 128 (8 KV heads, window 1024), 543 GFLOP, take 608 us call after call (584 at
// the least), 1.16 M cycles at a clock that falls to 1.9 GHz and below, of which
// the MFMAs are 49 %. A step of a SIMD's two waves takes 1.29 k cycles by
// itself, 1.02 k of them MFMAs, with the rounds' barriers and copies 1.55 k, and
// a workgroup's beginning and end are a fifth of its time. Without copies it is
// 11 % less, without LDS reads 3, without exponentials nothing; fragments read
// over the barrier, a fifth fewer scalar instructions and workgroups that start
// apart gave 0 to 3 % of cycles and no time. The steps on the way: scores and
// product of one block in turn 676 us, one block ahead and behind 670, queries
// and outputs through LDS and the hidden slots by a mask of bits 629, copies in
// assembly 618, values' fragments before the keys' 600 to 608. 16 ragged
// requests, 2860 tokens, heads of 64, 5 rounds each, are bound by latency: 16.7
// us.
// ---------------------------------------------------------------------------

template <typename T, int HD, int PARTS>
__global__ __launch_bounds__(PARTS == 1 ? 256 : 512, PARTS == 1 && HD == 64 ? 3 : 2) void window_tile_kernel(WindowArgs a) {
  constexpr int IMG = 2 * kKeys * HD;  // bytes of an image of 32 keys
  constexpr int GROUPS = PARTS == 1 ? 4 : 2, ROWS = 32 * GROUPS;   // of 32 rows, a wave of each part
  constexpr int BLOCKS = PARTS == 1 ? 2 : 1, ROUND = 32 * BLOCKS;  // of 32 keys; keys of a part's round
  constexpr int COPY = ROUND / GROUPS;                             // of which a wave copies
  __shared__ __attribute__((aligned(16))) uint8_t lds[PARTS][2][2][BLOCKS * IMG];  // [part][K, V][round & 1]
  __shared__ __attribute__((aligned(16))) uint8_t extra[PARTS == 1 ? IMG : 16];
  const nemo_attention_batch& b = a.b;
  const int kvh = blockIdx.x % a.kv_heads, tile_no = blockIdx.x / a.kv_heads;  // an XCD's L2 keeps to one KV head of 8
  const Request<ROWS> r(a, tile_no);
  if (r.i < 0) return;
  const int rows = r.queries * a.group, row0 = (tile_no - r.tile) * ROWS;
  if ((unsigned)row0 >= (unsigned)rows) return;
  const Heads<T> heads(a, r.q0, r.kv0, kvh);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hl = lane >> 5;
  const int behind = r.keys - r.queries;  // position of query 0
  const KeyList list(a, behind + a.query(row0), behind + a.query(min(row0 + ROWS - 1, rows - 1)), r.keys);
  const int group = wave % GROUPS, part = wave / GROUPS;
  const int w0 = row0 + 32 * group, w1 = min(w0 + 31, rows - 1);
  const int row = min(w0 + (lane & 31), rows - 1);  // (a wave past the rows takes the last one's)
  auto window = [&](int at) { return list.window(a, behind + a.query(at), r.keys); };
  const Seen mine = window(row), first = window(min(w0, rows - 1)), last = window(w1);
  const int rounds = (list.n + ROUND * PARTS - 1) / (ROUND * PARTS), base = ROUND * rounds * part;

  // A wave copies COPY rows of K and of V a round, of one of the two images of
  // each. V's first image of round `at` is the block before the round's, of
  // round 0 zeros.
  const int64_t k_stride = 2 * b.k_row, v_stride = 2 * b.v_row;
  const int second = COPY * group / 32;
  const Stager<HD, COPY, false> ks(COPY * group % 32, k_stride);
  const Stager<HD, COPY, true> vs(COPY * group % 32, v_stride);
  auto v_image = [&](int odd) { return lds[part][1][odd] + COPY * group * 2 * HD; };
  auto k_image = [&](int odd) { return lds[part][0][odd] + COPY * group * 2 * HD; };
  auto v_range = [&](int at) {
    const int t0 = base + ROUND * at - 32 + 32 * second;
    return vs.range((const uint8_t*)heads.v + list.key(t0) * v_stride, v_stride, t0 < base ? 0 : list.rows(t0));
  };
  auto k_range = [&](int at) {
    const int t0 = base + ROUND * at + 32 + 32 * second;
    return ks.range((const uint8_t*)heads.k + list.key(t0) * k_stride, k_stride, list.rows(t0));
  };
  Rows<T, HD> acc;
  acc.clear();
  float16v s;
  auto hidden = [&](int t0) {
    if (t0 + 32 > first.hi || (t0 < last.lo && t0 + 32 > a.sinks)) {
      asm volatile("");
      hide(s, t0, hl, mine.lo, mine.hi, a.sinks);
    }
  };
  // K of the first block; the group's queries, of which each part copies some
  uint8_t* const first_k = PARTS == 1 ? extra : lds[part][0][1];
  uint8_t* const rows_image = PARTS == 1 ? lds[0][group >> 1][1] + (group & 1) * IMG : lds[group][1][1];
  if (rounds) {
    const Stager<HD, 32 / GROUPS, false> k0(32 / GROUPS * group, k_stride);
    k0.copy(k0.range((const uint8_t*)heads.k + list.key(base) * k_stride, k_stride, list.rows(base)),
            first_k + 32 / GROUPS * group * 2 * HD);
    image_rows<HD>(lane, [&](int i, int r, int chunk) {
      if (i % PARTS != part) return;
      const int at = min(w0 + r, rows - 1);
      copy_address(heads.query(at, a.query(at)) + 8 * (chunk ^ k_swizzle<HD>(r)), rows_image + 1024 * i);
    });
    vs.copy(v_range(0), v_image(0));
    ks.copy(k_range(0), k_image(0));
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(IMG / 1024) : "memory");
    meet();
    acc.load(rows_image, lane);
    s = acc.scores(first_k, lane);
    hidden(base);
  }
  typename Mma<T>::frag p[2] = {};
  const bool tail = rounds && base + ROUND * rounds - 32 < list.n;  // the last round's last block has slots
  auto landed = [&] {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    meet();  // the round has landed, and every wave has left the other buffers
  };
  auto steps = [&](int at, const uint8_t* v_at, const uint8_t* k_at, auto&& copies) {
#pragma unroll
    for (int k = 0; k < BLOCKS; ++k) {
      acc.step(s, p, v_at + k * IMG, k_at + k * IMG, lane, a.scale2, [&](int c) { copies(HD / 16 * k + c); });
      hidden(base + ROUND * at + 32 + 32 * k);
    }
  };
  // (No round behind the last is staged but as zeros, which nobody reads.)
  for (int at = 0; at < rounds; at += 2) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (at + u >= rounds) break;
      landed();
      const u32x4 v = v_range(at + u + 1), k = k_range(at + u + 1);
      steps(at + u, lds[part][1][u], lds[part][0][u], [&](int c) {
        constexpr int N = HD / 32;  // copies of each
        if (c < N) vs.copy(v, c, v_image(1 - u));
        else if (c < 2 * N) ks.copy(k, c - N, k_image(1 - u));
      });
    }
  }
  if (rounds && ROUND * rounds - 32 < list.n) landed();  // (for the first part, so for all)
  if (tail) acc.values(lds[part][1][rounds & 1], lane, p);
  acc.l += __shfl_xor(acc.l, 32, 64);
  if constexpr (PARTS > 1) {
    // The other parts' sums go to the first's waves, each register as its 64 lanes.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    meet();
    auto sums = [&](int from) { return (float4v*)((uint8_t*)lds + (GROUPS * (from - 1) + group) * 2 * IMG) + lane; };
    auto ml = [&](int from) {
      return (float2*)((uint8_t*)lds + GROUPS * (PARTS - 1) * 2 * IMG) + 64 * (GROUPS * (from - 1) + group) + lane;
    };
    if (part) {
      *ml(part) = make_float2(acc.m, acc.l);
#pragma unroll
      for (int db = 0; db < HD / 32; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          sums(part)[64 * (4 * db + j)] =
              float4v{acc.o[db][4 * j], acc.o[db][4 * j + 1], acc.o[db][4 * j + 2], acc.o[db][4 * j + 3]};
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    meet();
    if (part) return;
    // (a part that saw nothing has the maximum -infinity and zeros)
    auto weight = [](float m, float most) { return m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - most); };
    float most = acc.m;
#pragma unroll
    for (int k = 1; k < PARTS; ++k) most = fmaxf(most, ml(k)->x);
    const float f = weight(acc.m, most);
    acc.l *= f;
#pragma unroll
    for (int db = 0; db < HD / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc.o[db][r] *= f;
#pragma unroll
    for (int k = 1; k < PARTS; ++k) {
      const float w = weight(ml(k)->x, most);
      acc.l = fmaf(w, ml(k)->y, acc.l);
#pragma unroll
      for (int db = 0; db < HD / 32; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4v v = sums(k)[64 * (4 * db + j)];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc.o[db][4 * j + e] = fmaf(w, v[e], acc.o[db][4 * j + e]);
        }
    }
  }
  // The list is that of all rows of the tile, and a value that some of them do
  // not see meets their probability 0; where it is not finite, their sums are
  // not, and they are taken again. (The rows of a tile of one query see every
  // key of the list. Those of a wave of one query need not.)
  const bool one_query = a.query(row0) == a.query(min(row0 + ROWS - 1, rows - 1));
  const uint64_t bad = one_query ? 0 : __builtin_amdgcn_ballot_w64(acc.spoilt());
  uint32_t again = (uint32_t)(bad | bad >> 32);
  if (again && !hidden_spoil<T, HD>(a, heads, list, first, last, 0, list.n)) again = 0;
  // Outputs go through LDS: whole rows to memory, 16 bytes a lane.
  if constexpr (PARTS == 1) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    meet();
  }
  uint8_t* const out_image = PARTS == 1 ? rows_image : (uint8_t*)lds + (4 * PARTS * BLOCKS - GROUPS + group) * IMG;
  acc.store((T*)(out_image + (lane & 31) * 2 * HD), lane & 31, hl);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  image_rows<HD>(lane, [&](int i, int r, int chunk) {
    const u32x4 v = *(const u32x4*)(out_image + r * 2 * HD + 16 * (chunk ^ k_swizzle<HD>(r)));
    if (w0 + r < rows && !(again >> r & 1)) *(u32x4*)(heads.output(w0 + r, a.query(w0 + r)) + 8 * chunk) = v;
  });
  for (uint32_t todo = again; todo; todo &= todo - 1) {
    const int at = w0 + __builtin_ctz(todo);
    if (at < rows) one_row<T, HD>(a, heads, list, r.queries, r.keys, at, 0, list.n).store(heads.output(at, a.query(at)));
  }
}

// ---------------------------------------------------------------------------
// Few rows: the 8 waves of a workgroup take the same 32 rows and every eighth
// block of 32 keys each, staged by the wave for itself (no barrier in the
// loop), and add up in LDS. A wave's next K is copied while it works on V, its
// next V while it works on K. With `splits` above 1 the blocks are dealt out
// to that many workgroups as well, whose sums a second kernel joins.
//
// Bound by memory where the caches are long: 64 tokens over 983 MB of keys and
// values 173 us (5.7 TB/s), one over 131072 keys 95 us and its join 4.6; by
// latency below: one token over 1028 keys of 64 8.6 us, of which the lookup,
// first loads and sums are about three quarters. With 4 waves it took 11.7.
// ---------------------------------------------------------------------------

constexpr int kFewWaves = 8;

// Sums of a split: the row's reference maximum and sum, and its output values.
struct Partials {
  float2* ml;  // [split][row], null: not split
  float* o;    // [split][row][HD]
  int64_t rows;
  int splits;
};

template <typename T, int HD>
__global__ __launch_bounds__(64 * kFewWaves) void window_few_kernel(WindowArgs a, Partials part) {
  constexpr int IMG = 2 * kKeys * HD;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kFewWaves][2 * IMG];  // K, V; later the waves' sums
  __shared__ float2 sums[kFewWaves][32];
  __shared__ uint32_t spoilt;
  // The float4 at column 4 c of a wave's row of sums.
  auto sum_at = [&](int wave, int row, int c) {
    return (float4v*)lds + (wave * 32 + row) * (HD / 4) + (c ^ (row & 15));
  };
  const nemo_attention_batch& b = a.b;
  const int kvh = blockIdx.x % a.kv_heads, tile_no = blockIdx.x / a.kv_heads, split = blockIdx.y;
  const Request<32> r(a, tile_no);
  if (r.i < 0) return;
  const int rows = r.queries * a.group, row0 = (tile_no - r.tile) * 32;
  if ((unsigned)row0 >= (unsigned)rows) return;
  const Heads<T> heads(a, r.q0, r.kv0, kvh);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hl = lane >> 5;
  const int behind = r.keys - r.queries, row1 = min(row0 + 31, rows - 1);
  const KeyList list(a, behind + a.query(row0), behind + a.query(row1), r.keys);
  const int row = min(row0 + (lane & 31), rows - 1);
  auto window = [&](int at) { return list.window(a, behind + a.query(at), r.keys); };
  const Seen mine = window(row), first = window(row0), last = window(row1);
  const int blocks = (list.n + 31) >> 5;
  const int block0 = (int)((int64_t)blocks * split / part.splits);
  const int block1 = (int)((int64_t)blocks * (split + 1) / part.splits);

  const int64_t k_stride = 2 * b.k_row, v_stride = 2 * b.v_row;
  const Stager<HD, 32, false> ks(0, k_stride);
  const Stager<HD, 32, true> vs(0, v_stride);
  uint8_t* const image = lds[wave];
  auto stage_k = [&](int at) {
    if (at >= block1) return;
    ks.copy(ks.range((const uint8_t*)heads.k + list.key(32 * at) * k_stride, k_stride, list.rows(32 * at)), image);
  };
  auto stage_v = [&](int at) {
    if (at >= block1) return;
    vs.copy(vs.range((const uint8_t*)heads.v + list.key(32 * at) * v_stride, v_stride, list.rows(32 * at)),
            image + IMG);
  };
  Rows<T, HD> acc;
  acc.clear();
  int at = block0 + wave;
  if (at < block1) {
    // the rows' image, where V goes next
    image_rows<HD>(lane, [&](int i, int r, int chunk) {
      const int qrow = min(row0 + r, rows - 1);
      copy_address(heads.query(qrow, a.query(qrow)) + 8 * (chunk ^ k_swizzle<HD>(r)), image + IMG + 1024 * i);
    });
    stage_k(at);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(IMG / 1024) : "memory");
    acc.load(image + IMG, lane);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    stage_v(at);
  }
  for (; at < block1; at += kFewWaves) {
    const int t0 = 32 * at;
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(IMG / 1024) : "memory");  // K, not yet V
    float16v s = acc.scores(image, lane);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    stage_k(at + kFewWaves);
    if (t0 + 32 > first.hi || (t0 < last.lo && t0 + 32 > a.sinks)) hide(s, t0, hl, mine.lo, mine.hi, a.sinks);
    typename Mma<T>::frag p[2];
    acc.exponentials(s, a.scale2, acc.m, p);
    acc.settle(s, a.scale2, p);
    if (at + kFewWaves < block1)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(IMG / 1024) : "memory");  // V, not yet the next K
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    acc.values(image + IMG, lane, p);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    stage_v(at + kFewWaves);
  }
  // The waves' sums: row-major in LDS, in place of the keys.
  acc.l += __shfl_xor(acc.l, 32, 64);
  if (threadIdx.x == 0) spoilt = 0;
  __syncthreads();
  if (row0 + (lane & 31) < rows) {
    if (hl == 0) sums[wave][lane] = make_float2(acc.m, acc.l);
#pragma unroll
    for (int db = 0; db < HD / 32; ++db)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4v v = {acc.o[db][4 * j], acc.o[db][4 * j + 1], acc.o[db][4 * j + 2], acc.o[db][4 * j + 3]};
        *sum_at(wave, lane & 31, 8 * db + 2 * j + hl) = v;
      }
  }
  __syncthreads();
  // Thread: C columns of one row.
  constexpr int C = HD / (2 * kFewWaves);
  const int mrow = threadIdx.x / (2 * kFewWaves), c0 = threadIdx.x % (2 * kFewWaves) * C;
  const bool valid = row0 + mrow < rows;
  float m = -INFINITY, l = 0.f, v[C] = {};
  if (valid) {
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) m = fmaxf(m, sums[w][mrow].x);
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
      const float2 ml = sums[w][mrow];
      if (ml.x == -INFINITY && ml.y == 0.f) continue;  // saw nothing
      const float f = ml.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - m);
      l = fmaf(f, ml.y, l);
#pragma unroll
      for (int c = 0; c < C; c += 4) {
        const float4v o = *sum_at(w, mrow, (c0 + c) / 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[c + e] = fmaf(f, o[e], v[c + e]);
      }
    }
    if (a.query(row0) != a.query(row1)) {
      float z = l * 0.f;
#pragma unroll
      for (int c = 0; c < C; ++c) z = fmaf(v[c], 0.f, z);
      if (z != 0.f) atomicOr(&spoilt, 1u << mrow);
    }
  }
  __syncthreads();
  const int64_t out_row = (int64_t)r.q0 * a.kv_heads * a.group + kvh * a.group;  // of row 0's first head, [query][head]
  auto partial = [&](int at) {
    const int i = a.query(at);
    return part.rows * split + out_row + (int64_t)i * a.kv_heads * a.group + (at - i * a.group);
  };
  uint32_t again = spoilt;
  if (again && !hidden_spoil<T, HD>(a, heads, list, first, last, 32 * block0, 32 * block1)) again = 0;
  if (valid && !(again >> mrow & 1)) {
    if (part.ml) {
      const int64_t at = partial(row0 + mrow);
      if (c0 == 0) part.ml[at] = make_float2(m, l);
#pragma unroll
      for (int c = 0; c < C; c += 4) *(float4v*)(part.o + at * HD + c0 + c) = float4v{v[c], v[c + 1], v[c + 2], v[c + 3]};
    } else {
      typedef T vec __attribute__((ext_vector_type(C)));
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      vec t;
#pragma unroll
      for (int c = 0; c < C; ++c) t[c] = (T)(v[c] * inv);
      *(vec*)(heads.output(row0 + mrow, a.query(row0 + mrow)) + c0) = t;
    }
  }
  // As in window_tile_kernel: rows spoilt by values that they do not see.
  uint32_t todo = again;
  for (int n = 0; todo; todo &= todo - 1, ++n) {
    if (n % kFewWaves != wave) continue;
    const int at = row0 + __builtin_ctz(todo);
    const OneRow<T, HD> one = one_row<T, HD>(a, heads, list, r.queries, r.keys, at, 32 * block0, min(32 * block1, list.n));
    if (part.ml) {
      if (lane == 0) part.ml[partial(at)] = make_float2(one.m, one.l);
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) part.o[partial(at) * HD + lane + 64 * c] = one.o[c];
    } else {
      one.store(heads.output(at, a.query(at)));
    }
  }
}

// Joins the splits, at most 64: a workgroup a row. Thread (g, c) adds columns 4
// c.. of splits g, g + G, ..., and the G sums are added in order.
template <typename T, int HD>
__global__ __launch_bounds__(256) void window_join_kernel(WindowArgs a, Partials part) {
  constexpr int C = HD / 4, G = 256 / C;
  __shared__ float weight[64];
  __shared__ float4v sums[G][C];
  const nemo_attention_batch& b = a.b;
  const int kvh = blockIdx.x % a.kv_heads, tile_no = blockIdx.x / a.kv_heads;
  const Request<1> r(a, tile_no);
  if (r.i < 0) return;
  const int row = tile_no - r.tile, lane = threadIdx.x & 63;
  if ((unsigned)row >= (unsigned)(r.queries * a.group)) return;
  const int i = a.query(row), h = kvh * a.group + (row - i * a.group);
  const int64_t at = (int64_t)(r.q0 + i) * a.kv_heads * a.group + h;
  // every wave: lane z's split
  const float2 ml = lane < part.splits ? part.ml[part.rows * lane + at] : make_float2(-INFINITY, 0.f);
  float m = ml.x;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
  const bool empty = ml.x == -INFINITY && ml.y == 0.f;  // saw nothing; its values mean nothing
  const float f = empty ? 0.f : ml.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - m);
  float l = empty ? 0.f : f * ml.y;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) l += __shfl_xor(l, x, 64);
  if (threadIdx.x < 64) weight[lane] = empty ? -1.f : f;
  __syncthreads();
  const int c = threadIdx.x % C, g = threadIdx.x / C;
  float4v v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int z = g; z < part.splits; z += G) {
    const float4v o = *(const float4v*)(part.o + (part.rows * z + at) * HD + 4 * c);
    const float w = weight[z];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = w == -1.f ? v[e] : fmaf(w, o[e], v[e]);
  }
  sums[g][c] = v;
  __syncthreads();
  if (threadIdx.x >= HD) return;
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < G; ++k) sum += sums[k][threadIdx.x / 4][threadIdx.x % 4];
  T* out = (T*)b.out + (int64_t)(r.q0 + i) * b.out_row + h * b.out_head;
  out[threadIdx.x] = (T)(l == 0.f ? 0.f : sum / l);
}

__global__ __launch_bounds__(256) void ragged_index_kernel(Ragged rows, int64_t* __restrict__ positions,
                                                           int32_t* __restrict__ q_start,
                                                           int64_t* __restrict__ kv_start,
                                                           int32_t* __restrict__ kv_len) {
  const int t = blockIdx.x * 256 + threadIdx.x, total = rows.start[rows.count];
  if (t < total) {
    int b = 0;
    while (t >= rows.start[b + 1]) ++b;
    positions[t] = t - rows.start[b];
  }
  if (t <= rows.count) q_start[t] = rows.start[t];
  if (t < rows.count) {
    kv_start[t] = rows.start[t];
    kv_len[t] = rows.start[t + 1] - rows.start[t];
  }
}

// Which kernel a batch takes and how its keys are split, by its sizes alone.
// `tiles` of 32 rows, of which window_few_kernel has `places` on the chip at a
// time, and the keys that a query sees; microseconds few : tile : tile of 4
// parts, 32 heads, 8 KV heads.
//  Tiles that fit: few (64: 500 tokens +-128 9.2 : 9.0, 512 of a 512-key window
//  10.6 : 12.0; 128: 250 tokens of a 512-key window 10.1 : 15.4 : 13.2, 256
//  behind 8192 keys 52 : 134 : 74).
//  More, requests of at most 8 rows, whose keys come from memory: few from 512
//  keys and 1.5 to 8 times the places (single tokens, heads of 128, 2052 keys:
//  36 of them 76 : 68, 44 81 : 76, 52 84 : 84, 96 141 : 164, 256 370 : 386, 512
//  735 : 749; 132 keys: 96 23 : 19.6; heads of 64: 104 97 : 110, 320 260 : 280,
//  1024 830 : 783), else tile, as for more rows (64 x 4 tokens, heads of 128 117
//  : 99; 64 x 8 131 : 101).
//  More than twice as many: tile (64: 2000 tokens +-128 28 : 13.8; 128: 520
//  tokens, 1024 keys 33 : 23.6 : 32.4).
//  Between, heads of 128 whose tiles of 64 rows fit: 4 parts from 384 keys (500
//  tokens of 132 keys 14.8 : 9.7 : 10.8, 260 15.9 : 11.6 : 12.2, 516 18.6 : 15.6
//  : 13.6, 1028 23.4 : 23.6 : 17.7; 4 x 128, 1028 keys 24.4 : 24.5 : 20.2).
//  Between, larger requests, heads of 64: few up to 1.5 places from 2048 keys
//  (1028 keys: 600 tokens 18.5 : 18.5; 2052: 600 27.5 : 31.5, 800 33.2 : 31.4;
//  8600: 600 80 : 110); else tile.
// A split costs a second launch, 3.5 us, and is taken from 1280 keys (single
// token, heads of 64, unsplit : split: 1100 keys 8.3 : 9.4, 1800 10.5 : 9.4,
// 8000 33.6 : 11.0), into pieces of 256 keys and more for more rows, whose sums
// are written and read again (8 tokens over 8192 keys of 128: pieces of 256
// 20.6, of 512 15.7).
struct Plan {
  enum { kFew, kTile, kParts } kernel;
  int splits;
};
Plan window_plan(const nemo_attention_config& c, int count, int64_t q_rows, int64_t max_kv) {
  if (count == 0 || q_rows == 0) return {Plan::kTile, 1};
  const int64_t rows = q_rows * (c.q_heads / c.kv_heads);
  auto tiles_of = [&](int n) { return std::max<int64_t>(rows / n, count) * c.kv_heads; };
  const int64_t tiles = tiles_of(32), places = c.head_dim == 64 ? 512 : 256;
  int64_t keys = max_kv;
  if (c.left >= 0 && c.right >= 0) keys = std::min(keys, (int64_t)c.left + c.right + 1 + c.sinks);
  if (tiles > places) {
    if (rows / count <= 8)
      return {keys >= 512 && 2 * tiles >= 3 * places && tiles <= 8 * places ? Plan::kFew : Plan::kTile, 1};
    if (tiles > 2 * places) return {Plan::kTile, 1};
    if (c.head_dim == 128 && tiles_of(64) <= places && keys >= 384) return {Plan::kParts, 1};
    return {c.head_dim == 64 && 2 * tiles <= 3 * places && keys >= 2048 ? Plan::kFew : Plan::kTile, 1};
  }
  const int64_t piece = 256 + 8 * std::min<int64_t>(32, rows / count);
  const int64_t splits = keys < 1280 ? 1 : std::min<int64_t>({places / tiles, keys / piece, 64});
  return {Plan::kFew, (int)std::max<int64_t>(1, splits)};
}

}  // namespace

size_t window_workspace(const nemo_attention_config& c, int count, int64_t q_rows, int64_t max_kv) {
  const int splits = window_plan(c, count, q_rows, max_kv).splits;
  return splits == 1 ? 0 : (size_t)splits * q_rows * c.q_heads * (c.head_dim * 4 + 8);
}

hipError_t launch_ragged_index(const Ragged& rows, int64_t* positions, int32_t* q_start, int64_t* kv_start,
                               int32_t* kv_len, hipStream_t stream) {
  const int n = std::max(rows.start[rows.count], rows.count + 1);
  ragged_index_kernel<<<(n + 255) / 256, 256, 0, stream>>>(rows, positions, q_start, kv_start, kv_len);
  return hipGetLastError();
}

hipError_t launch_window_attention(const nemo_attention_config& c, const nemo_attention_batch& b, hipStream_t stream) {
  if (b.count == 0 || b.q_rows == 0) return hipSuccess;
  WindowArgs a{b, c.kv_heads, c.q_heads / c.kv_heads, 0, 0, 0, 0.f, 0, 0};
  // Copies' ranges end one stride behind a row's start; that of a single row may be anything.
  if (b.kv_rows == 1) a.b.k_row = a.b.v_row = c.head_dim;
  while (1 << a.shift < a.group) ++a.shift;
  a.magic = (uint32_t)((((uint64_t)1 << a.shift) - a.group) * ((uint64_t)1 << 32) / a.group + 1);
  auto bound = [](int v) { return v < 0 ? kUnbounded : std::min(v, kUnbounded); };
  a.left = bound(c.left);
  a.right = bound(c.right);
  a.sinks = std::min(c.sinks, kUnbounded);
  a.scale2 = (c.scale > 0.f ? c.scale : 1.0f / sqrtf((float)c.head_dim)) * 1.4426950408889634f;
  const Plan plan = window_plan(c, b.count, b.q_rows, b.max_kv);
  const int splits = b.workspace ? plan.splits : 1;
  const int64_t rows = b.q_rows * c.q_heads;
  Partials part{nullptr, nullptr, rows, splits};
  if (splits > 1) {
    part.o = (float*)b.workspace;
    part.ml = (float2*)(part.o + splits * rows * c.head_dim);
  }
  auto tiles = [&](int r) { return (unsigned)(b.q_rows * a.group / r + b.count) * c.kv_heads; };
  auto launch = [&](auto type, auto hd) {
    constexpr int HD = decltype(hd)::value;
    typedef decltype(type) T;
    if (plan.kernel == Plan::kTile) {
      window_tile_kernel<T, HD, 1><<<tiles(128), 256, 0, stream>>>(a);
      return;
    }
    if constexpr (HD == 128) {
      if (plan.kernel == Plan::kParts) {
        window_tile_kernel<T, HD, 4><<<tiles(64), 512, 0, stream>>>(a);
        return;
      }
    }
    window_few_kernel<T, HD><<<dim3(tiles(32), splits), 64 * kFewWaves, 0, stream>>>(a, part);
    if (splits > 1) window_join_kernel<T, HD><<<tiles(1), 256, 0, stream>>>(a, part);
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
