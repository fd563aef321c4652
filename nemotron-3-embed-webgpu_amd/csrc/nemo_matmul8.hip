// Products of 8-bit rows and weights for gfx950 (include/nemo.h nemo_matmul8):
// y[i][j] = x_scale[i] w_scale[j] (sum over k of x[i][k] w[j][k]) + bias[j],
// the sum in 32-bit integers, exact, on v_mfma_i32_16x16x64_i8.
//
// Both operands of that instruction are 16 rows, lane l with bytes 16 (l / 16) ..
// + 15 of row l % 16, so rows are read as they lie, 16 bytes a lane. W is the
// first operand: a lane's four results are four neighbouring columns of a row
// of y.
#include <math.h>

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
  // Scales and biases of four columns. (Loaded before the first store, which
  // the compiler takes to change them.)
  struct Columns {
    float4v scale, bias;
  };
  __device__ __forceinline__ Columns columns(int j) const {
    Columns c;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = min(j + e, a.n - 1);
      c.scale[e] = a.w_scale[at];
      c.bias[e] = a.bias ? a.bias[at] : 0.f;
    }
    return c;
  }
  __device__ __forceinline__ float row(int64_t i) const { return a.x_scale[min(i, a.m - 1) * a.x_scale_row]; }
  // Sums of columns j .. j + 3 of row i.
  __device__ __forceinline__ void store(int64_t i, int j, int4v c, float scale, const Columns& of) const {
    if (i >= a.m || j >= a.n) return;
    T* y = (T*)a.y + i * a.y_row + j;
    T v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (T)((float)c[e] * scale * of.scale[e] + of.bias[e]);
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
// Few tiles: a workgroup takes 16 MT rows of x and 16 NT rows of W, its 8 waves
// blocks of 128 k in turn, each copied into images of the wave's own (no barrier
// in the loop), and adds up in LDS. (Fragments loaded from memory take a
// quarter of the rate, 16 bytes a cycle and CU: neighbouring lanes have
// neighbouring rows. 77 x 2048 x 6144 took 13.3 us that way, 6.9 this way.)
// Workgroups begin at different blocks, since rows a power of two apart lie on
// few channels of memory (1 x 8192 x 8192, 16 x 32 18.4 -> 12.2).
//
// One row is bound by memory and the launch: 5120 x 2048, 10.5 MB, 3.8 us; 8192 x
// 8192, 67 MB, 12.1 (5.5 TB/s); between, by LDS and L2: each byte of an image
// is written and read once.
// ---------------------------------------------------------------------------

constexpr int kWaves = 8;

template <typename T, int MT, int NT, int STAGES>
__global__ __launch_bounds__(64 * kWaves) void matmul8_few_kernel(nemo_matmul8_args a, int tiles_n) {
  constexpr int WAVES = kWaves, TILES = MT * NT, STEP = TILES < 8 ? TILES : 8, C = 2 * (MT + NT), IMG = 1024 * C;
  static_assert(STEP * 1024 <= STAGES * IMG, "sums fit");
  __shared__ __attribute__((aligned(16))) uint8_t lds[WAVES][STAGES * IMG];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile_n = blockIdx.x % tiles_n, n0 = tile_n * 16 * NT;
  const int64_t m0 = (int64_t)(blockIdx.x / tiles_n) * 16 * MT;
  const int whole = (a.k + 3) & ~3, wr = min(16 * NT, a.n - n0), xr = (int)min((int64_t)16 * MT, a.m - m0);
  const int64_t w_row = a.n > 1 ? a.w_row : whole, x_row = a.m > 1 ? a.x_row : whole;
  const int8_t *x = a.x + m0 * x_row, *w = a.w + n0 * w_row;
  const int64_t x_bytes = (xr - 1) * x_row + whole, w_bytes = (wr - 1) * w_row + whole;
  const uint32_t chunk = 16 * ((lane & 7) ^ (lane >> 3));
  uint32_t x_at[2 * MT], w_at[2 * NT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) x_at[i] = (uint32_t)((8 * i + (lane >> 3)) * x_row) + chunk;
#pragma unroll
  for (int i = 0; i < 2 * NT; ++i) w_at[i] = (uint32_t)((8 * i + (lane >> 3)) * w_row) + chunk;
  const int blocks = (a.k + 127) >> 7, begin = blocks ? 2 * (tile_n >> 3) % blocks : 0;
  auto block = [&](int i) { return i + begin < blocks ? i + begin : i + begin - blocks; };
  // (Blocks behind the last are copied as zeros, which nobody reads: the waits count copies.)
  auto copy = [&](int i, const uint8_t* to) {
    const int64_t at = 128 * (int64_t)(i < blocks ? block(i) : 0);
    const u32x4 xs = range_of(x + at, i < blocks ? (uint32_t)(x_bytes - at) : 0);
    const u32x4 ws = range_of(w + at, i < blocks ? (uint32_t)(w_bytes - at) : 0);
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) copy_range(ws, w_at[i], to + 1024 * i);
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) copy_range(xs, x_at[i], to + 2048 * NT + 1024 * i);
  };
  int4v c[NT][MT] = {};
  uint8_t* const ring = lds[wave];
#pragma unroll
  for (int i = 0; i < STAGES; ++i) copy(wave + WAVES * i, ring + IMG * i);
  const int row = lane & 15;
  int stage = 0;
  for (int i = wave; i < blocks; i += WAVES) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * C) : "memory");
    const uint8_t* at = ring + IMG * stage + 128 * row;
    u32x4 wv[2][NT], xv[2][MT];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int k = 16 * ((4 * s + (lane >> 4)) ^ (row & 7));
#pragma unroll
      for (int t = 0; t < NT; ++t) wv[s][t] = *(const u32x4*)(at + 2048 * t + k);
#pragma unroll
      for (int t = 0; t < MT; ++t) xv[s][t] = *(const u32x4*)(at + 2048 * (NT + t) + k);
    }
    const int b = block(i);
    if (128 * b + 128 > a.k) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int t = 0; t < MT; ++t) xv[s][t] = row_end(xv[s][t], 128 * b + 64 * s + 16 * (lane >> 4), a.k);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    copy(i + STAGES * WAVES, ring + IMG * stage);
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) c[n][m] = mma(wv[s][n], xv[s][m], c[n][m]);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  const Out<T> out(a);
#pragma unroll
  for (int from = 0; from < TILES; from += STEP) {
    if (from) __syncthreads();
#pragma unroll
    for (int t = 0; t < STEP; ++t)
      if (from + t < TILES) ((int4v*)ring)[64 * t + lane] = c[(from + t) / MT][(from + t) % MT];
    __syncthreads();
    for (int t = wave; t < STEP && from + t < TILES; t += WAVES) {
      int4v s = ((const int4v*)lds[0])[64 * t + lane];
#pragma unroll
      for (int i = 1; i < WAVES; ++i) s += ((const int4v*)lds[i])[64 * t + lane];
      const int64_t i = m0 + 16 * ((from + t) % MT) + (lane & 15);
      const int j = n0 + 16 * ((from + t) / MT) + 4 * (lane >> 4);
      out.store(i, j, s, out.row(i), out.columns(j));
    }
  }
}

// ---------------------------------------------------------------------------
// Tiles of BM rows of x and BN rows of W: WM x WN waves, STAGES blocks of 128 k
// in LDS, copied by DMA. A row of an image is 8 chunks of 16 bytes, chunk c of row
// r at c ^ (r % 8): the 16 rows of a fragment lie on all banks. A half block's
// fragments are read among the products of the half before, whose order is
// pinned (left to itself the compiler puts the reads behind the products); the
// barrier of a block stands between its halves, where no wave waits for LDS, and
// frees the block for the copies that follow it.
//
// Bound by the matrix cores and the clock, which falls to about 2 GHz under them:
// 16384 x 8192 x 8192 in 880 us is 2.50 PFLOP/s (a library's product of these bytes,
// without scales, 902), 2400 x 12288 x 2048 in 67 is 1.79. On the way: fragments
// read before their products, tiles column by column 1013 and 91; 8 row tiles
// side by side, reads of a half ahead 976 and 93; scales loaded before the
// stores 914 and 75; the order pinned 880 and 69.
// ---------------------------------------------------------------------------

template <typename T, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(64 * WM * WN) void matmul8_tile_kernel(nemo_matmul8_args a, int tiles_n, int tiles) {
  constexpr int WAVES = WM * WN, MT = BM / WM / 16, NT = BN / WN / 16;
  constexpr int XC = BM / 8 / WAVES, WC = BN / 8 / WAVES;  // copies of 8 rows by a wave
  __shared__ __attribute__((aligned(16))) int8_t lds[STAGES][(BM + BN) * 128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // an XCD (workgroup i is on XCD i % 8) takes tiles that follow each other, 8 row
  // tiles side by side: what its CUs read at a time fits its L2 several times over
  constexpr int group = 8;
  const int q = tiles >> 3, r = tiles & 7, xcd = blockIdx.x & 7;
  const int tile = xcd * q + min(xcd, r) + (blockIdx.x >> 3);
  const int tiles_m = tiles / tiles_n, of = tile / (group * tiles_n), in = tile - of * group * tiles_n;
  const int high = min(group, tiles_m - of * group);
  const int64_t m0 = (int64_t)(of * group + in % high) * BM;
  const int n0 = in / high * BN;
  const int whole = (a.k + 3) & ~3, wr = min(BN, a.n - n0), xr = (int)min((int64_t)BM, a.m - m0);
  const int64_t w_row = a.n > 1 ? a.w_row : whole, x_row = a.m > 1 ? a.x_row : whole;
  const int8_t *x = a.x + m0 * x_row, *w = a.w + n0 * w_row;
  const int64_t x_bytes = (xr - 1) * x_row + whole, w_bytes = (wr - 1) * w_row + whole;
  const uint32_t chunk = 16 * ((lane & 7) ^ (lane >> 3));
  uint32_t x_at[XC], w_at[WC];
#pragma unroll
  for (int i = 0; i < XC; ++i) x_at[i] = (uint32_t)((8 * (XC * wave + i) + (lane >> 3)) * x_row) + chunk;
#pragma unroll
  for (int i = 0; i < WC; ++i) w_at[i] = (uint32_t)((8 * (WC * wave + i) + (lane >> 3)) * w_row) + chunk;
  const int blocks = (a.k + 127) >> 7;
  // (Blocks behind the last are copied as zeros, which nobody reads: the waits count copies.)
  struct Block {
    u32x4 x, w;
  };
  auto block = [&](int b) {
    const int64_t at = 128 * (int64_t)b;
    return Block{range_of(x + at, b < blocks ? (uint32_t)(x_bytes - at) : 0),
                 range_of(w + at, b < blocks ? (uint32_t)(w_bytes - at) : 0)};
  };
  auto copy = [&](const Block& from, int i, int8_t* to) {
    if (i < XC) copy_range(from.x, x_at[i], (const uint8_t*)to + 1024 * (XC * wave + i));
    else copy_range(from.w, w_at[i - XC], (const uint8_t*)to + 128 * BM + 1024 * (WC * wave + i - XC));
  };
  const int wm = wave % WM, wn = wave / WM, row = lane & 15, quarter = lane >> 4;
  int4v c[NT][MT] = {};
  // Fragments of 64 k, read one by one.
  struct Half {
    u32x4 x[MT], w[NT];
  };
  constexpr int READS = MT + NT, PRODUCTS = MT * NT, COPIES = XC + WC;
  auto read = [&](Half& f, const int8_t* from, int half, int i) {
    const int at = 16 * ((4 * half + quarter) ^ (row & 7));
    if (i < NT) f.w[i] = *(const u32x4*)(from + (BM + 16 * (NT * wn + i) + row) * 128 + at);
    else f.x[i - NT] = *(const u32x4*)(from + (16 * (MT * wm + i - NT) + row) * 128 + at);
  };
  auto mask = [&](Half& f, int half) {
#pragma unroll
    for (int t = 0; t < MT; ++t) f.x[t] = row_end(f.x[t], 128 * (blocks - 1) + 64 * half + 16 * quarter, a.k);
  };
  // Products of a half, with other instructions among them: each(i) behind the i-th.
  auto products = [&](const Half& f, auto&& each) {
#pragma unroll
    for (int i = 0; i < PRODUCTS; ++i) {
      c[i / MT][i % MT] = mma(f.w[i / MT], f.x[i % MT], c[i / MT][i % MT]);
      each(i);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int i = 0; i < STAGES; ++i) {
    const Block from = block(i);
#pragma unroll
    for (int j = 0; j < COPIES; ++j) copy(from, j, lds[i]);
  }
  Half first, second;
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * COPIES) : "memory");
  meet();
#pragma unroll
  for (int i = 0; i < READS; ++i) read(first, lds[0], 0, i);
  int stage = 0;
  const int full = a.k >> 7;
  for (int b = 0; b < full; ++b) {
    // (a READS-th of the products between two reads at most)
    products(first, [&](int i) {
#pragma unroll
      for (int r = 0; r < READS; ++r)
        if (r * (PRODUCTS / 2) / READS == i) read(second, lds[stage], 1, r);
    });
    // the next block has landed, and every wave has read this one
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * COPIES) : "memory");
    meet();
    __builtin_amdgcn_sched_barrier(0);
    const int next = stage + 1 == STAGES ? 0 : stage + 1;
    const Block from = block(b + STAGES);
    products(second, [&](int i) {
#pragma unroll
      for (int r = 0; r < READS; ++r)
        if (r * (PRODUCTS / 2) / READS == i) read(first, lds[next], 0, r);
#pragma unroll
      for (int j = 0; j < COPIES; ++j)
        if (j * PRODUCTS / COPIES == i) copy(from, j, lds[stage]);
    });
    stage = next;
  }
  if (full < blocks) {
    mask(first, 0);
#pragma unroll
    for (int i = 0; i < READS; ++i) read(second, lds[stage], 1, i);
    products(first, [](int) {});
    mask(second, 1);
    products(second, [](int) {});
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the LDS is another workgroup's afterwards
  const Out<T> out(a);
  auto column = [&](int t) { return n0 + 16 * (NT * wn + t) + 4 * quarter; };
  auto row_of = [&](int t) { return m0 + 16 * (MT * wm + t) + row; };
  typename Out<T>::Columns columns[NT];
  float scales[MT];
#pragma unroll
  for (int t = 0; t < NT; ++t) columns[t] = out.columns(column(t));
#pragma unroll
  for (int j = 0; j < MT; ++j) scales[j] = out.row(row_of(j));
#pragma unroll
  for (int j = 0; j < MT; ++j)
#pragma unroll
    for (int t = 0; t < NT; ++t) out.store(row_of(j), column(t), c[t][j], scales[j], columns[t]);
}

// A variant's tile, and its price, to be compared with the others': in microseconds of
// what 33 sizes of 1 to 8192 rows, 700 to 12288 columns and 100 to 8192 k took: `begin`,
// and `step` for each 128 k
// and four times for the sums' way out, as often as its workgroups have to
// follow each other on 256 CUs; `whole`: in whole rounds. (No time where all CUs work for
// long and the clock falls: 8192 x 8192 x 8192 is priced at 317 and takes 455.) Over the 33 the
// choice takes 1 % more than the fastest on average (few kernel of 16 x 16, 16 x 32,
// 32 x 32, 32 x 64 : tiles of 64 x 64, 128 x 64, 256 x 128, 256 x 256; 1 x 2048 x
// 6144 4.6, 5.7, 6.2, 8.2 : 11.6; 77 x 2048 x 6144 9.7, 9.0, 6.9, 9.4 : 12.3; 150 x 5120
// x 2048 10.2, 9.4 of the last two : 6.9, 10.5; 1024 x 2048 x 2048 19.2, 18.6 : 10.2,
// 10.9, 17.4; 1500 x 4096 x 4096 42.5, 40.8, 30.6, 46.7 of the tiles; 2400 x 12288 x 2048
// 109, 98, 81, 67).
struct Variant {
  int rows, columns;
  bool whole;
  double begin, step;
};
constexpr Variant kVariants[] = {
    {16, 16, true, 1.9, 0.072},  {16, 32, true, 1.95, 0.082},  {32, 32, true, 1.85, 0.12},
    {32, 64, true, 1.4, 0.2},    {64, 64, false, 2.7, 0.198},  {128, 64, false, 2.95, 0.319},
    {256, 128, true, 4.6, 0.57}, {256, 256, true, 5.8, 1.08},
};
constexpr int kVariantCount = sizeof(kVariants) / sizeof(*kVariants);
int variant_of(int64_t m, int64_t n, int k) {
  int best = kVariantCount - 1;
  double least = INFINITY;
  for (int i = 0; i < kVariantCount; ++i) {
    const Variant& v = kVariants[i];
    const double groups = (double)((m + v.rows - 1) / v.rows) * (double)((n + v.columns - 1) / v.columns);
    if (groups >= 0x1p22 && i != kVariantCount - 1) continue;  // (grids hold less than 2^32 threads)
    const double rounds = v.whole ? ceil(groups / 256) : fmax(1.0, groups / 256);
    const double time = rounds * v.step * (k / 128.0 + 4) + v.begin * (v.rows >= 256 ? rounds : 1.0);
    if (time < least) {
      best = i;
      least = time;
    }
  }
  return best;
}

}  // namespace

hipError_t launch_matmul8(const nemo_matmul8_args& a, hipStream_t stream) {
  if (a.m == 0 || a.n == 0) return hipSuccess;
  auto typed = [&](auto type) {
    typedef decltype(type) T;
    auto few = [&](auto mt, auto nt, auto stages) {
      constexpr int MT = decltype(mt)::value, NT = decltype(nt)::value;
      const int tn = (a.n + 16 * NT - 1) / (16 * NT), all = (int)((a.m + 16 * MT - 1) / (16 * MT)) * tn;
      matmul8_few_kernel<T, MT, NT, decltype(stages)::value><<<all, 64 * kWaves, 0, stream>>>(a, tn);
    };
    auto tiles = [&](auto bm, auto bn, auto wm, auto wn, auto stages) {
      constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WM = decltype(wm)::value,
                    WN = decltype(wn)::value;
      const int tn = (a.n + BN - 1) / BN, all = (int)((a.m + BM - 1) / BM) * tn;
      matmul8_tile_kernel<T, BM, BN, WM, WN, decltype(stages)::value><<<all, 64 * WM * WN, 0, stream>>>(a, tn, all);
    };
#define N(v) std::integral_constant<int, v>{}
    switch (variant_of(a.m, a.n, a.k)) {
      case 0: return few(N(1), N(1), N(2));
      case 1: return few(N(1), N(2), N(1));
      case 2: return few(N(2), N(2), N(1));
      case 3: return few(N(2), N(4), N(1));
      case 4: return tiles(N(64), N(64), N(2), N(2), N(4));
      case 5: return tiles(N(128), N(64), N(2), N(2), N(3));
      case 6: return tiles(N(256), N(128), N(2), N(4), N(3));
      default: return tiles(N(256), N(256), N(2), N(4), N(2));
    }
#undef N
  };
  if (a.type == NEMO_TYPE_F32) typed(float{});
  else if (a.type == NEMO_TYPE_F16) typed(half_t{});
  else typed(bf16_t{});
  return hipGetLastError();
}

}  // namespace nemo
