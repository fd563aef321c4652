// Products of 8-bit rows and weights for gfx950 (include/nemo.h nemo_matmul8):
// y[i][j] = x_scale[i] w_scale[j] (sum over k of x[i][k] w[j][k]) + bias[j],
// the sum in 32-bit integers, exact, on v_mfma_i32_16x16x64_i8.
//
// Both operands of that instruction are 16 rows, lane l with bytes 16 (l / 16) ..
// + 15 of row l % 16, so rows are read as they lie, 16 bytes a lane. W is the
// first operand: a lane's four results are four neighbouring columns of a row
// of y.
#include <algorithm>
#include <type_traits>

#include "nemo_lds_copy.h"
#include "nemo_operators.h"

namespace nemo {

namespace {

typedef int int4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int4v mma(u32x4 w, u32x4 x, int4v c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(int4v, w), __builtin_bit_cast(int4v, x), c, 0, 0, 0);
}

// A buffer of `bytes` bytes at `at`: loads past its end give zeros.
__device__ __forceinline__ u32x4 range_of(const int8_t* at, uint32_t bytes) {
  return u32x4{(uint32_t)(uintptr_t)at, (uint32_t)((uintptr_t)at >> 32) & 0xffffu,
               (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}
__device__ __forceinline__ u32x4 load_range(u32x4 range, uint32_t offset) {
  return __builtin_amdgcn_raw_buffer_load_b128(
      __builtin_amdgcn_make_buffer_rsrc((void*)((uint64_t)range[1] << 32 | range[0]), 0, range[2], 0x00020000), offset,
      0, 0);
}

// 16 bytes of a row from byte `at` on, without those past the row's end.
__device__ __forceinline__ u32x4 row_end(u32x4 v, int at, int k) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = min(max(k - at - 4 * i, 0), 4);
    v[i] &= n == 4 ? ~0u : (1u << (8 * n)) - 1;
  }
  return v;
}

template <typename T>
struct Out {
  const nemo_matmul8_args& a;
  bool vectors;  // four values of a row may be stored as one
  __device__ __forceinline__ Out(const nemo_matmul8_args& args) : a(args) {
    vectors = ((uintptr_t)a.y & (4 * sizeof(T) - 1)) == 0 && a.y_row % 4 == 0;
  }
  // Sums of columns j .. j + 3 of row i < m.
  __device__ __forceinline__ void store(int64_t i, int j, int4v c) const {
    T* y = (T*)a.y + i * a.y_row + j;
    const float s = a.x_scale[i * a.x_scale_row];
    T v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = min(j + e, a.n - 1);
      const float t = (float)c[e] * s * a.w_scale[at];
      v[e] = (T)(a.bias ? t + a.bias[at] : t);
    }
    if (vectors && j + 4 <= a.n) {
      typedef T vec __attribute__((ext_vector_type(4)));
      *(vec*)y = vec{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j + e < a.n) y[e] = v[e];
    }
  }
};

// ---------------------------------------------------------------------------
// Few rows of x: a workgroup takes 16 rows of W and all 16 MT rows of x, its 8
// waves blocks of 256 k in turn, whose sums they add in LDS. W goes from memory to
// registers.
// ---------------------------------------------------------------------------

constexpr int kSkinnyWaves = 8;

template <typename T, int MT>
__global__ __launch_bounds__(64 * kSkinnyWaves) void matmul8_skinny_kernel(nemo_matmul8_args a) {
  __shared__ int4v sums[kSkinnyWaves][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
  const int whole = (a.k + 3) & ~3, wr = min(16, a.n - n0);
  const int64_t w_row = a.n > 1 ? a.w_row : 0, x_row = a.m > 1 ? a.x_row : 0;
  const int xr = (int)min((int64_t)16 * MT, a.m - m0);
  const u32x4 w = range_of(a.w + n0 * w_row, (uint32_t)((wr - 1) * w_row + whole));
  const u32x4 x = range_of(a.x + m0 * x_row, (uint32_t)((xr - 1) * x_row + whole));
  const uint32_t w_at = min(lane & 15, wr - 1) * (uint32_t)w_row;
  uint32_t x_at[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) x_at[t] = min(16 * t + (lane & 15), xr - 1) * (uint32_t)x_row;
  int4v c[MT] = {};
  const int blocks = (a.k + 255) >> 8;
  for (int b = wave; b < blocks; b += kSkinnyWaves) {
    const int k0 = 256 * b + 16 * (lane >> 4);
    u32x4 wv[4], xv[MT][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) wv[i] = load_range(w, w_at + k0 + 64 * i);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) xv[t][i] = load_range(x, x_at[t] + k0 + 64 * i);
    if (256 * b + 256 > a.k) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) xv[t][i] = row_end(xv[t][i], k0 + 64 * i, a.k);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < MT; ++t) c[t] = mma(wv[i], xv[t][i], c[t]);
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) sums[wave][t][lane] = c[t];
  __syncthreads();
  const Out<T> out(a);
#pragma unroll
  for (int t = 0; t < MT; t += kSkinnyWaves) {
    if (t + wave >= MT) break;
    int4v s = sums[0][t + wave][lane];
#pragma unroll
    for (int i = 1; i < kSkinnyWaves; ++i) s += sums[i][t + wave][lane];
    const int64_t i = m0 + 16 * (t + wave) + (lane & 15);
    if (i < a.m && n0 + 4 * (lane >> 4) < a.n) out.store(i, n0 + 4 * (lane >> 4), s);
  }
}

// ---------------------------------------------------------------------------
// Tiles of BM rows of x and BN rows of W: WM x WN waves, blocks of 128 k copied
// into LDS, one block ahead. A row of an image is 8 chunks of 16 bytes, chunk c
// of row r at c ^ (r % 8): the 16 rows of a fragment lie on all banks.
// ---------------------------------------------------------------------------

template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void matmul8_tile_kernel(nemo_matmul8_args a, int tiles_n, int tiles) {
  constexpr int WAVES = WM * WN, MT = BM / WM / 16, NT = BN / WN / 16;
  constexpr int XC = BM / 8 / WAVES, WC = BN / 8 / WAVES;  // copies of 8 rows by a wave
  __shared__ __attribute__((aligned(16))) int8_t lds[2][(BM + BN) * 128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // an XCD (workgroup i is on XCD i % 8) takes tiles that follow each other, column by column
  const int q = tiles >> 3, r = tiles & 7, xcd = blockIdx.x & 7;
  const int tile = xcd * q + min(xcd, r) + (blockIdx.x >> 3);
  const int tiles_m = tiles / tiles_n;
  const int64_t m0 = (int64_t)(tile % tiles_m) * BM;
  const int n0 = tile / tiles_m * BN;
  const int whole = (a.k + 3) & ~3, wr = min(BN, a.n - n0), xr = (int)min((int64_t)BM, a.m - m0);
  const int64_t w_row = a.n > 1 ? a.w_row : whole, x_row = a.m > 1 ? a.x_row : whole;
  const int8_t *x = a.x + m0 * x_row, *w = a.w + n0 * w_row;
  const uint32_t x_bytes = (uint32_t)((xr - 1) * x_row + whole), w_bytes = (uint32_t)((wr - 1) * w_row + whole);
  const uint32_t chunk = 16 * ((lane & 7) ^ (lane >> 3));
  uint32_t x_at[XC], w_at[WC];
#pragma unroll
  for (int i = 0; i < XC; ++i) x_at[i] = (uint32_t)((8 * (XC * wave + i) + (lane >> 3)) * x_row) + chunk;
#pragma unroll
  for (int i = 0; i < WC; ++i) w_at[i] = (uint32_t)((8 * (WC * wave + i) + (lane >> 3)) * w_row) + chunk;
  const int blocks = (a.k + 127) >> 7;
  auto copy = [&](int b, int8_t* to) {
    const u32x4 xs = range_of(x + 128 * b, x_bytes - 128 * b), ws = range_of(w + 128 * b, w_bytes - 128 * b);
#pragma unroll
    for (int i = 0; i < XC; ++i) copy_range(xs, x_at[i], (const uint8_t*)to + 1024 * (XC * wave + i));
#pragma unroll
    for (int i = 0; i < WC; ++i) copy_range(ws, w_at[i], (const uint8_t*)to + 128 * BM + 1024 * (WC * wave + i));
  };
  const int wm = wave % WM, wn = wave / WM, row = lane & 15;
  int4v c[NT][MT] = {};
  if (blocks) copy(0, lds[0]);
  for (int b = 0; b < blocks; ++b) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    meet();  // the block has landed, and every wave has left the other one
    if (b + 1 < blocks) copy(b + 1, lds[(b + 1) & 1]);
    const int8_t *xs = lds[b & 1] + (16 * MT * wm + row) * 128, *ws = lds[b & 1] + (BM + 16 * NT * wn + row) * 128;
    const bool end = 128 * b + 128 > a.k;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int at = 16 * ((4 * s + (lane >> 4)) ^ (row & 7));
      u32x4 xv[MT], wv[NT];
#pragma unroll
      for (int t = 0; t < MT; ++t) xv[t] = *(const u32x4*)(xs + 16 * 128 * t + at);
#pragma unroll
      for (int t = 0; t < NT; ++t) wv[t] = *(const u32x4*)(ws + 16 * 128 * t + at);
      if (end) {
#pragma unroll
        for (int t = 0; t < MT; ++t) xv[t] = row_end(xv[t], 128 * b + 64 * s + 16 * (lane >> 4), a.k);
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) c[i][j] = mma(wv[i], xv[j], c[i][j]);
    }
  }
  const Out<T> out(a);
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int64_t i = m0 + 16 * (MT * wm + j) + row;
    if (i >= a.m) continue;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int n = n0 + 16 * (NT * wn + t) + 4 * (lane >> 4);
      if (n < a.n) out.store(i, n, c[t][j]);
    }
  }
}

}  // namespace

hipError_t launch_matmul8(const nemo_matmul8_args& a, hipStream_t stream) {
  if (a.m == 0 || a.n == 0) return hipSuccess;
  auto typed = [&](auto type) {
    typedef decltype(type) T;
    if (a.m <= 64) {
      const unsigned grid = (a.n + 15) / 16;
      if (a.m <= 16) matmul8_skinny_kernel<T, 1><<<grid, 64 * kSkinnyWaves, 0, stream>>>(a);
      else if (a.m <= 32) matmul8_skinny_kernel<T, 2><<<grid, 64 * kSkinnyWaves, 0, stream>>>(a);
      else matmul8_skinny_kernel<T, 4><<<grid, 64 * kSkinnyWaves, 0, stream>>>(a);
      return;
    }
    auto tiles = [&](auto bm, auto bn, auto wm, auto wn) {
      constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WM = decltype(wm)::value,
                    WN = decltype(wn)::value;
      const int tn = (a.n + BN - 1) / BN, all = (int)((a.m + BM - 1) / BM) * tn;
      matmul8_tile_kernel<T, BM, BN, WM, WN><<<all, 64 * WM * WN, 0, stream>>>(a, tn, all);
    };
    using std::integral_constant;
    if ((a.m + 255) / 256 * ((a.n + 255) / 256) >= 256)
      tiles(integral_constant<int, 256>{}, integral_constant<int, 256>{}, integral_constant<int, 2>{}, integral_constant<int, 4>{});
    else
      tiles(integral_constant<int, 128>{}, integral_constant<int, 128>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
  };
  if (a.type == NEMO_TYPE_F32) typed(float{});
  else if (a.type == NEMO_TYPE_F16) typed(half_t{});
  else typed(bf16_t{});
  return hipGetLastError();
}

}  // namespace nemo
