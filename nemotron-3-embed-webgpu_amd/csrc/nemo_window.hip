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

#include "nemo_operators.h"

namespace nemo {

namespace {

struct WindowArgs {
  nemo_attention_batch b;
  int kv_heads, group, left, right, sinks;
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
  static __device__ __forceinline__ float16v mma(frag a, frag b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<bf16_t> {
  typedef bf16x8 frag;
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

// Copies of ROWS key rows into an image by one wave, 1 KB an instruction:
// rows first .. first + ROWS of a 32-row image (or of two that follow each
// other). lane_off: the lane's byte offsets from the address of slot row 0 of
// the image, for rows that lie `stride` bytes apart.
template <int HD, int ROWS, bool VALUES>
struct Stager {
  static constexpr int kChunks = HD / 8, kPer = 64 / kChunks, kN = ROWS / kPer;
  uint32_t off[kN];
  int row, chunk[kN];
  __device__ __forceinline__ Stager(int first, int64_t stride) {
    const int lane = threadIdx.x & 63;
    row = first + lane / kChunks;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int r = row + kPer * i;
      chunk[i] = 16 * ((lane % kChunks) ^ (VALUES ? v_swizzle<HD>(r) : k_swizzle<HD>(r)));
      off[i] = (uint32_t)(r * stride) + chunk[i];
    }
  }
  // Slots t0 .. of the list, all of them window keys: consecutive rows from `at`.
  __device__ __forceinline__ void rows(const uint8_t* at, uint8_t* image) const {
#pragma unroll
    for (int i = 0; i < kN; ++i)
      __builtin_amdgcn_global_load_lds((const void*)(at + off[i]), (lds_void*)(image + 1024 * i), 16, 0, 0);
  }
  // Any slots: key(t) of each, the last slot's from there on.
  template <typename Key>
  __device__ __forceinline__ void slots(const uint8_t* base, int64_t stride, int t0, int n, Key&& key,
                                        uint8_t* image) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int64_t j = key(min(t0 + row + kPer * i, n - 1));
      __builtin_amdgcn_global_load_lds((const void*)(base + j * stride + chunk[i]), (lds_void*)(image + 1024 * i), 16,
                                       0, 0);
    }
  }
};

// The tile of 32 rows of a wave, or the larger one of a workgroup: its key
// list, and in list coordinates what the row of a lane sees: t < hi and (t >= lo
// or t < sinks).
struct KeyList {
  int sinks, lo, n;  // slots t < sinks are keys t, others lo + t - sinks
  __device__ __forceinline__ KeyList(const WindowArgs& a, int p0, int p1, int keys) {
    const Seen first(a, p0, keys), last(a, p1, keys);
    lo = first.lo;
    sinks = min(a.sinks, lo);
    n = sinks + last.hi - lo;
  }
  __device__ __forceinline__ int key(int t) const { return t < sinks ? t : lo + t - sinks; }
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
  float m, l;

  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
  }
  __device__ __forceinline__ void load(const T* row, int hl) {
#pragma unroll
    for (int c = 0; c < DC; ++c) q[c] = *(const frag*)(row + 16 * c + 8 * hl);
  }
  __device__ __forceinline__ float16v scores(const uint8_t* image, int lane) const {
    const int row = lane & 31, hl = lane >> 5, sw = k_swizzle<HD>(row);
    float16v s = {};
#pragma unroll
    for (int c = 0; c < DC; ++c)
      s = Mma<T>::mma(*(const frag*)(image + row * 2 * HD + 16 * ((2 * c + hl) ^ sw)), q[c], s);
    return s;
  }
  // Probabilities against a reference maximum that is raised only when a row
  // exceeds it by 2^8 (a wave vote): p <= 256 then, far from overflow, and
  // most blocks need no exchange between lanes and no rescaling; numerator
  // and denominator share the reference, so the result is the softmax. A row
  // that has seen nothing yet has the reference 0.
  __device__ __forceinline__ void probabilities(const float16v& s, float scale2, frag (&p)[2]) {
    float most = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) most = fmaxf(most, s[r]);
    most *= scale2;
    if (__builtin_amdgcn_ballot_w64(most > m + 8.0f)) {
      asm volatile("");  // keeps the rare path a branch
      const float mn = fmaxf(m, fmaxf(most, __shfl_xor(most, 32, 64)));
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
      l *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
      m = mn;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    float e[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      e[r] = __builtin_amdgcn_exp2f(fmaf(s[r], scale2, -ref));
      l += e[r];
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float8v f;
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = e[8 * c + i];
      p[c] = __builtin_convertvector(f, frag);
    }
  }
  // O^T += V^T P^T: k slot 8 hl + e of chunk c is key 16 c + 8 (e / 4) + 4 hl + e
  // % 4, score register 8 c + e. A transposed read gives the 16 lanes of a
  // group 4 keys of 16 columns; lane i of it reads key i / 4's columns 4 (i % 4)...
  __device__ __forceinline__ void values(const uint8_t* image, int lane, const frag (&p)[2]) {
    const int i = lane & 15, hl = lane >> 5;
    const int key = 4 * hl + (i >> 2), half = (lane >> 4) & 1;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const int chunk = 4 * db + 2 * half + ((i >> 1) & 1);
        short8v a;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int r = 16 * c + 8 * u + key;
          const short4v v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_short4v*)(image + r * 2 * HD + 16 * (chunk ^ v_swizzle<HD>(r)) + 8 * (i & 1)));
#pragma unroll
          for (int e = 0; e < 4; ++e) a[4 * u + e] = v[e];
        }
        o[db] = Mma<T>::mma(__builtin_bit_cast(frag, a), p[c], o[db]);
      }
  }
  __device__ __forceinline__ void store(T* out, int hl) const {
    typedef T vec __attribute__((ext_vector_type(4)));
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        vec v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(o[db][4 * j + e] * inv);
        *(vec*)(out + 32 * db + 8 * j + 4 * hl) = v;
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

// Scores of hidden slots of the block at t0 become -infinity.
__device__ __forceinline__ void hide(float16v& s, int t0, int hl, int lo, int hi, int sinks) {
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int t = t0 + 8 * (r >> 2) + 4 * hl + (r & 3);
    if (!(t < hi && (t >= lo || t < sinks))) s[r] = -INFINITY;
  }
}

// Addresses of one request and KV head.
template <typename T>
struct Heads {
  const T *q, *k, *v;
  T* out;
  int64_t q_row, q_head, out_row, out_head;
  int group;
  __device__ __forceinline__ Heads(const WindowArgs& a, const Request& r, int kvh)
      : q_row(a.b.q_row), q_head(a.b.q_head), out_row(a.b.out_row), out_head(a.b.out_head), group(a.group) {
    q = (const T*)a.b.q + r.q0 * q_row + (int64_t)kvh * group * q_head;
    k = (const T*)a.b.k + r.kv0 * a.b.k_row + kvh * a.b.k_head;
    v = (const T*)a.b.v + r.kv0 * a.b.v_row + kvh * a.b.v_head;
    out = (T*)a.b.out + r.q0 * out_row + (int64_t)kvh * group * out_head;
  }
  __device__ __forceinline__ const T* query(int row) const {
    return q + (row / group) * q_row + (row % group) * q_head;
  }
  __device__ __forceinline__ T* output(int row) const {
    return out + (row / group) * out_row + (row % group) * out_head;
  }
};

// A row over the slots [t0, t1) that it sees, key by key.
template <typename T, int HD>
__device__ __forceinline__ OneRow<T, HD> one_row(const WindowArgs& a, const Heads<T>& h, const KeyList& list,
                                                 const Request& r, int row, int t0, int t1) {
  const Seen seen(a, r.keys - r.queries + row / h.group, r.keys);
  const int lo = seen.lo - list.lo + list.sinks, hi = seen.hi - list.lo + list.sinks, first = min(a.sinks, hi);
  OneRow<T, HD> acc;
  acc.keys(h.query(row), h.k, a.b.k_row, h.v, a.b.v_row, t0, min(t1, first), a.scale2);
  const int from = max(max(t0, lo), first), to = min(t1, hi);
  if (from < to) acc.keys(h.query(row), h.k, a.b.k_row, h.v, a.b.v_row, list.key(from), list.key(to - 1) + 1, a.scale2);
  return acc;
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup of 4 waves takes 128 rows, 32 a wave, and stages 64
// keys a round for all of them, two rounds deep.
// ---------------------------------------------------------------------------

constexpr int kTileRows = 128;

template <typename T, int HD>
__global__ __launch_bounds__(256, HD == 128 ? 2 : 4) void window_tile_kernel(WindowArgs a) {
  constexpr int IMG = 2 * kKeys * HD;  // bytes of an image of 32 keys
  __shared__ __attribute__((aligned(16))) uint8_t lds[2][4 * IMG];  // [stage]: K, K, V, V
  const nemo_attention_batch& b = a.b;
  const int kvh = blockIdx.x % a.kv_heads, tile_no = blockIdx.x / a.kv_heads;  // an XCD's L2 keeps to one KV head of 8
  const int request = tile_request(b, a.group, kTileRows, tile_no);
  if (request < 0) return;
  const Request r(b, request);
  const int rows = r.queries * a.group, row0 = (tile_no - tile_base(b, a.group, kTileRows, request)) * kTileRows;
  if (row0 >= rows) return;
  const Heads<T> heads(a, r, kvh);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hl = lane >> 5;
  const int behind = r.keys - r.queries;  // position of query 0
  const KeyList list(a, behind + row0 / a.group, behind + min(row0 + kTileRows - 1, rows - 1) / a.group, r.keys);
  const int w0 = row0 + 32 * wave, w1 = min(w0 + 31, rows - 1);
  const bool active = w0 < rows;
  const int row = min(w0 + (lane & 31), rows - 1);
  auto window = [&](int at) {
    Seen s(a, behind + at / a.group, r.keys);
    s.lo += list.sinks - list.lo;
    s.hi += list.sinks - list.lo;
    return s;
  };
  const Seen mine = window(row), first = window(min(w0, rows - 1)), last = window(w1);
  const int rounds = (list.n + 63) >> 6;

  const int64_t k_stride = 2 * b.k_row, v_stride = 2 * b.v_row;
  const Stager<HD, 16, false> ks(16 * wave, k_stride);
  const Stager<HD, 16, true> vs(16 * wave, v_stride);
  auto stage = [&](int at) {
    uint8_t* ki = lds[at & 1] + 16 * wave * 2 * HD;
    uint8_t* vi = ki + 2 * IMG;
    const int t0 = 64 * at;
    if (t0 >= list.sinks && t0 + 64 <= list.n) {
      const int64_t j = list.key(t0);
      ks.rows((const uint8_t*)heads.k + j * k_stride, ki);
      vs.rows((const uint8_t*)heads.v + j * v_stride, vi);
    } else {
      auto key = [&](int t) { return list.key(t); };
      ks.slots((const uint8_t*)heads.k, k_stride, t0, list.n, key, ki);
      vs.slots((const uint8_t*)heads.v, v_stride, t0, list.n, key, vi);
    }
  };
  if (rounds) stage(0);
  Rows<T, HD> acc;
  acc.load(heads.query(row), hl);
  acc.clear();
  for (int at = 0; at < rounds; ++at) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // this round has landed, and every wave has left the other stage
    if (at + 1 < rounds) stage(at + 1);
    if (!active) continue;
    const uint8_t* image = lds[at & 1];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t0 = 64 * at + 32 * u;
      if (t0 >= last.hi || (t0 + 32 <= first.lo && t0 >= a.sinks)) continue;  // no row sees it
      float16v s = acc.scores(image + u * IMG, lane);
      if (t0 + 32 > first.hi || (t0 < last.lo && t0 + 32 > a.sinks)) hide(s, t0, hl, mine.lo, mine.hi, a.sinks);
      typename Mma<T>::frag p[2];
      acc.probabilities(s, a.scale2, p);
      acc.values(image + (2 + u) * IMG, lane, p);
    }
  }
  if (!active) return;
  acc.l += __shfl_xor(acc.l, 32, 64);
  // A value that some rows of the wave do not see meets their probability 0;
  // where it is not finite, their sums are not, and they are taken again. (One
  // query's rows see the same keys.)
  const uint64_t bad = w0 / a.group == w1 / a.group ? 0 : __builtin_amdgcn_ballot_w64(acc.spoilt());
  const uint32_t again = (uint32_t)(bad | bad >> 32);
  if (w0 + (lane & 31) < rows && !(again >> (lane & 31) & 1)) acc.store(heads.output(row), hl);
  for (uint32_t todo = again; todo; todo &= todo - 1) {
    const int at = w0 + __builtin_ctz(todo);
    if (at < rows) one_row<T, HD>(a, heads, list, r, at, 0, list.n).store(heads.output(at));
  }
}

// ---------------------------------------------------------------------------
// Few rows: the 4 waves of a workgroup take the same 32 rows and every fourth
// block of 32 keys each, staged by the wave for itself two blocks deep (no
// barrier in the loop), and add up in LDS. With `splits` above 1 the blocks are
// dealt out to that many workgroups as well, whose sums a second kernel joins.
// ---------------------------------------------------------------------------

constexpr int kFewWaves = 4;

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
  constexpr int OP = HD + 4;  // row of the sums in LDS, in floats
  __shared__ __attribute__((aligned(16))) uint8_t lds[kFewWaves][2][2 * IMG];
  __shared__ float2 sums[kFewWaves][32];
  __shared__ uint32_t spoilt;
  static_assert(kFewWaves * 32 * OP * 4 <= sizeof(lds), "the sums fit in the keys' place");
  const nemo_attention_batch& b = a.b;
  const int kvh = blockIdx.x % a.kv_heads, tile_no = blockIdx.x / a.kv_heads, split = blockIdx.y;
  const int request = tile_request(b, a.group, 32, tile_no);
  if (request < 0) return;
  const Request r(b, request);
  const int rows = r.queries * a.group, row0 = (tile_no - tile_base(b, a.group, 32, request)) * 32;
  if (row0 >= rows) return;
  const Heads<T> heads(a, r, kvh);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hl = lane >> 5;
  const int behind = r.keys - r.queries, row1 = min(row0 + 31, rows - 1);
  const KeyList list(a, behind + row0 / a.group, behind + row1 / a.group, r.keys);
  const int row = min(row0 + (lane & 31), rows - 1);
  auto window = [&](int at) {
    Seen s(a, behind + at / a.group, r.keys);
    s.lo += list.sinks - list.lo;
    s.hi += list.sinks - list.lo;
    return s;
  };
  const Seen mine = window(row), first = window(row0), last = window(row1);
  const int blocks = (list.n + 31) >> 5;
  const int block0 = (int)((int64_t)blocks * split / part.splits);
  const int block1 = (int)((int64_t)blocks * (split + 1) / part.splits);

  const int64_t k_stride = 2 * b.k_row, v_stride = 2 * b.v_row;
  const Stager<HD, 32, false> ks(0, k_stride);
  const Stager<HD, 32, true> vs(0, v_stride);
  auto stage = [&](int at, int buffer) {
    uint8_t* ki = lds[wave][buffer];
    const int t0 = 32 * at;
    if (t0 >= list.sinks && t0 + 32 <= list.n) {
      const int64_t j = list.key(t0);
      ks.rows((const uint8_t*)heads.k + j * k_stride, ki);
      vs.rows((const uint8_t*)heads.v + j * v_stride, ki + IMG);
    } else {
      auto key = [&](int t) { return list.key(t); };
      ks.slots((const uint8_t*)heads.k, k_stride, t0, list.n, key, ki);
      vs.slots((const uint8_t*)heads.v, v_stride, t0, list.n, key, ki + IMG);
    }
  };
  Rows<T, HD> acc;
  acc.load(heads.query(row), hl);
  acc.clear();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the queries: from here on only copies are counted
  int at = block0 + wave;
  if (at < block1) stage(at, 0);
  for (int buffer = 0; at < block1; at += kFewWaves, buffer ^= 1) {
    if (at + kFewWaves < block1) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the other buffer's reads are done
      stage(at + kFewWaves, buffer ^ 1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * IMG / 1024) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const int t0 = 32 * at;
    if (t0 >= last.hi || (t0 + 32 <= first.lo && t0 >= a.sinks)) continue;
    float16v s = acc.scores(lds[wave][buffer], lane);
    if (t0 + 32 > first.hi || (t0 < last.lo && t0 + 32 > a.sinks)) hide(s, t0, hl, mine.lo, mine.hi, a.sinks);
    typename Mma<T>::frag p[2];
    acc.probabilities(s, a.scale2, p);
    acc.values(lds[wave][buffer] + IMG, lane, p);
  }
  // The waves' sums: row-major in LDS, in place of the keys.
  acc.l += __shfl_xor(acc.l, 32, 64);
  if (threadIdx.x == 0) spoilt = 0;
  __syncthreads();
  float* o = (float*)lds;
  if (row0 + (lane & 31) < rows) {
    if (hl == 0) sums[wave][lane] = make_float2(acc.m, acc.l);
#pragma unroll
    for (int db = 0; db < HD / 32; ++db)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4v v = {acc.o[db][4 * j], acc.o[db][4 * j + 1], acc.o[db][4 * j + 2], acc.o[db][4 * j + 3]};
        *(float4v*)(o + (wave * 32 + (lane & 31)) * OP + 32 * db + 8 * j + 4 * hl) = v;
      }
  }
  __syncthreads();
  // Thread: HD / 8 columns of one row.
  constexpr int C = HD / 8;
  const int mrow = threadIdx.x >> 3, c0 = (threadIdx.x & 7) * C;
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
      for (int c = 0; c < C; ++c) v[c] = fmaf(f, o[(w * 32 + mrow) * OP + c0 + c], v[c]);
    }
    if (row0 / a.group != row1 / a.group) {
      float z = l * 0.f;
#pragma unroll
      for (int c = 0; c < C; ++c) z = fmaf(v[c], 0.f, z);
      if (z != 0.f) atomicOr(&spoilt, 1u << mrow);
    }
  }
  __syncthreads();
  const int64_t out_row = (int64_t)r.q0 * a.kv_heads * a.group + kvh * a.group;  // of row 0's first head, [query][head]
  auto partial = [&](int at) {
    return part.rows * split + out_row + (int64_t)(at / a.group) * a.kv_heads * a.group + at % a.group;
  };
  const uint32_t again = spoilt;
  if (valid && !(again >> mrow & 1)) {
    if (part.ml) {
      const int64_t at = partial(row0 + mrow);
      if (c0 == 0) part.ml[at] = make_float2(m, l);
#pragma unroll
      for (int c = 0; c < C; c += 4) *(float4v*)(part.o + at * HD + c0 + c) = float4v{v[c], v[c + 1], v[c + 2], v[c + 3]};
    } else {
      typedef T vec __attribute__((ext_vector_type(8)));
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      T* out = heads.output(row0 + mrow) + c0;
#pragma unroll
      for (int c = 0; c < C; c += 8) {
        vec t;
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = (T)(v[c + e] * inv);
        *(vec*)(out + c) = t;
      }
    }
  }
  // As in window_tile_kernel: rows spoilt by values that they do not see.
  uint32_t todo = again;
  for (int n = 0; todo; todo &= todo - 1, ++n) {
    if (n % kFewWaves != wave) continue;
    const int at = row0 + __builtin_ctz(todo);
    const OneRow<T, HD> one = one_row<T, HD>(a, heads, list, r, at, 32 * block0, min(32 * block1, list.n));
    if (part.ml) {
      if (lane == 0) part.ml[partial(at)] = make_float2(one.m, one.l);
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) part.o[partial(at) * HD + lane + 64 * c] = one.o[c];
    } else {
      one.store(heads.output(at));
    }
  }
}

// Joins the splits: a wave a row, lane z the weight of split z (at most 64).
template <typename T, int HD>
__global__ __launch_bounds__(256) void window_join_kernel(WindowArgs a, Partials part) {
  constexpr int R = 4;
  const nemo_attention_batch& b = a.b;
  const int kvh = blockIdx.x % a.kv_heads, tile_no = blockIdx.x / a.kv_heads;
  const int request = tile_request(b, a.group, R, tile_no);
  if (request < 0) return;
  const Request r(b, request);
  const int row = (tile_no - tile_base(b, a.group, R, request)) * R + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= r.queries * a.group) return;
  const int64_t at = (int64_t)(r.q0 + row / a.group) * a.kv_heads * a.group + kvh * a.group + row % a.group;
  const float2 ml = lane < part.splits ? part.ml[part.rows * lane + at] : make_float2(-INFINITY, 0.f);
  float m = ml.x;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
  const bool empty = ml.x == -INFINITY && ml.y == 0.f;
  const float f = empty ? 0.f : ml.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - m);
  float l = empty ? 0.f : f * ml.y;
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) l += __shfl_xor(l, x, 64);
  const uint64_t full = ~__builtin_amdgcn_ballot_w64(empty);
  float v[HD / 64] = {};
  for (int z = 0; z < part.splits; ++z) {
    if (!(full >> z & 1)) continue;
    const float fz = __shfl(f, z, 64);
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) v[c] = fmaf(fz, part.o[(part.rows * z + at) * HD + lane + 64 * c], v[c]);
  }
  T* out = (T*)b.out + (int64_t)(r.q0 + row / a.group) * b.out_row + (kvh * a.group + row % a.group) * b.out_head;
#pragma unroll
  for (int c = 0; c < HD / 64; ++c) out[lane + 64 * c] = (T)(l == 0.f ? 0.f : v[c] / l);
}

// Whether the keys are dealt out to the waves of a workgroup, not the rows:
// when tiles of 128 rows would leave CUs without one.
bool few_rows(const nemo_attention_config& c, int64_t q_rows) {
  return q_rows * c.q_heads < 256 * kTileRows;
}

}  // namespace

int window_splits(const nemo_attention_config& c, int count, int64_t q_rows, int64_t max_kv) {
  if (count == 0 || q_rows == 0 || !few_rows(c, q_rows)) return 1;
  const int64_t tiles = std::max<int64_t>(q_rows * (c.q_heads / c.kv_heads) / 32, count) * c.kv_heads;
  int64_t keys = max_kv;
  if (c.left >= 0 && c.right >= 0)
    keys = std::min(keys, (int64_t)c.left + c.right + c.sinks + (q_rows + count - 1) / count);
  return (int)std::max<int64_t>(1, std::min<int64_t>({(512 + tiles - 1) / tiles, keys / 256, 64}));
}

size_t window_workspace(const nemo_attention_config& c, int count, int64_t q_rows, int64_t max_kv) {
  const int splits = window_splits(c, count, q_rows, max_kv);
  return splits == 1 ? 0 : (size_t)splits * q_rows * c.q_heads * (c.head_dim * 4 + 8);
}

hipError_t launch_window_attention(const nemo_attention_config& c, const nemo_attention_batch& b, hipStream_t stream) {
  if (b.count == 0 || b.q_rows == 0) return hipSuccess;
  WindowArgs a{b, c.kv_heads, c.q_heads / c.kv_heads, 0, 0, 0, 0.f};
  auto bound = [](int v) { return v < 0 ? kUnbounded : std::min(v, kUnbounded); };
  a.left = bound(c.left);
  a.right = bound(c.right);
  a.sinks = std::min(c.sinks, kUnbounded);
  a.scale2 = (c.scale > 0.f ? c.scale : 1.0f / sqrtf((float)c.head_dim)) * 1.4426950408889634f;
  const int splits = b.workspace ? window_splits(c, b.count, b.q_rows, b.max_kv) : 1;
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
    if (!few_rows(c, b.q_rows)) {
      window_tile_kernel<T, HD><<<tiles(kTileRows), 256, 0, stream>>>(a);
      return;
    }
    window_few_kernel<T, HD><<<dim3(tiles(32), splits), 64 * kFewWaves, 0, stream>>>(a, part);
    if (splits > 1) window_join_kernel<T, HD><<<tiles(4), 256, 0, stream>>>(a, part);
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
