// Tiles of attention for gfx950: a wave's 32 rows against keys and values in LDS
// images of 32 keys, scores transposed and in registers.
#pragma once

#include <type_traits>

#include "nemo_operators.h"

namespace nemo {
namespace {

typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef float float8v __attribute__((ext_vector_type(8)));
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

// The rows of an image of 32, 16 bytes a lane: do(i, row, chunk) for row kPer i +
// lane / kChunks of the image and its chunk, i < HD / 16.
template <int HD, typename Do>
__device__ __forceinline__ void image_rows(int lane, Do&& each) {
  constexpr int kChunks = HD / 8, kPer = 64 / kChunks;
#pragma unroll
  for (int i = 0; i < kKeys / kPer; ++i) each(i, kPer * i + lane / kChunks, lane % kChunks);
}

}  // namespace
}  // namespace nemo
