// Matrix products of the int8 activations for MI355X (gfx950): the int8 product with scales per row and channel,
// and the weight gradient taken from an int8 checkpoint.

#include "int8_common.h"

namespace {

using namespace optimi_int8;

typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

#define OPTIMI_LDS __attribute__((address_space(3)))
#define OPTIMI_GLOBAL __attribute__((address_space(1)))

// 16 bytes per lane from global memory to LDS, past the registers.  The LDS side is `lds` (the same for the whole
// wave) plus 16 bytes per lane; the global side is `offset` bytes behind a buffer's base, a multiple of 16 per lane.
// The buffer's size bounds the access: lanes beyond it read nothing, and nobody uses what is in their place.
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer_of(const void* base, int64_t bytes) {
  const int64_t most = 0x7fffffff;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)(bytes < 0 ? 0 : bytes < most ? bytes : most), 0x00020000);
}
__device__ __forceinline__ void copy16_to_lds(Buffer from, uint32_t offset, void* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (OPTIMI_LDS void*)lds, 16, offset, 0, 0, 0);
}

__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64); }

// Consecutive workgroups go to the eight XCDs in turn, and each XCD has an L2 of its own.  An XCD gets a contiguous
// run of tiles instead, and runs walk the tiles in stripes of kStripe tile rows, so that the tiles in work on
// one XCD at a time form a patch that shares its operands' rows in L2.
constexpr int kXcds = 8;
constexpr int kStripe = 4;
struct Tile {
  int row, col;
};
__device__ __forceinline__ Tile tile_of(int id, int rows, int cols) {
  const int total = rows * cols, per = total / kXcds, more = total % kXcds;
  const int xcd = id % kXcds, at = id / kXcds;
  const int t = xcd * per + (xcd < more ? xcd : more) + at;
  const int stripe = t / (kStripe * cols), first = stripe * kStripe;
  const int height = rows - first < kStripe ? rows - first : kStripe;
  const int in = t - first * cols;
  return {first + in % height, in / height};
}

// The steps [begin, end) of a sum over two pairs of tiles in LDS: while one is multiplied, the next step's is on its
// way.  fetch<which>(step) starts the loads, settle<which>() finishes them and lets the workgroup meet, multiply<which>()
// adds the tile's products.  The last step's tile may end anywhere, so it has a fetch of its own that looks at every
// border, and its products leave out what is not there; the others' fetch needs no care.  The last step works on the first
// pair of tiles, and which pair the first step takes follows from that; the second pair is free when the sums are done.
template <int I>
using Pair = std::integral_constant<int, I>;
template <class Fetch, class FetchLast, class Settle, class Multiply, class MultiplyLast>
__device__ __forceinline__ void run_steps(int begin, int end, Fetch fetch, FetchLast fetch_last, Settle settle, Multiply multiply, MultiplyLast multiply_last) {
  const Pair<0> p0;
  const Pair<1> p1;
  if (begin >= end) return;
  if (end - begin == 1) {
    fetch_last(begin, p0);
    settle(p0);
    multiply_last(p0);
    return;
  }
  int step = begin;
  if ((end - begin) % 2) {
    fetch(step, p0);
    settle(p0);
    fetch(++step, p1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(p0);
    settle(p1);
  } else {
    fetch(step, p1);
    settle(p1);
  }
  for (; step + 2 < end; step += 2) {
    fetch(step + 1, p0);
    __builtin_amdgcn_sched_barrier(0);  // the loads start before the products do; left alone, they are moved behind them
    multiply(p1);
    settle(p0);
    fetch(step + 2, p1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(p0);
    settle(p1);
  }
  fetch_last(end - 1, p0);
  __builtin_amdgcn_sched_barrier(0);
  multiply(p1);
  settle(p0);
  multiply_last(p0);
}

// A wave's way from the matrix instruction's layout to rows: R rows of C 32-bit results in LDS, in pieces of four;
// the piece's place is mixed with the row so that neither side's accesses meet in one bank.
template <int R, int C>
struct OutBlock {
  static constexpr int kBytes = R * C * 4;
  static constexpr int kLanes = C / 8;            // lanes of a row, eight results each
  static constexpr int kTurns = R * kLanes / 64;  // rows that a lane has
  static __device__ __forceinline__ int col() { return threadIdx.x % 64 % kLanes * 8; }
  static __device__ __forceinline__ int row(int turn) { return turn * (64 / kLanes) + threadIdx.x % 64 / kLanes; }
  static __device__ __forceinline__ int at(int row, int piece) { return row * C + ((piece ^ (row & 7)) * 4); }
  static __device__ __forceinline__ void put(uint32_t* block, int row, int piece, u32x4 v) { *(u32x4*)(block + at(row, piece)) = v; }
  static __device__ __forceinline__ void get(const uint32_t* block, int row, uint32_t (&v)[8]) {
    const u32x4 lo = *(const u32x4*)(block + at(row, col() / 4)), hi = *(const u32x4*)(block + at(row, col() / 4 + 1));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = lo[e];
      v[4 + e] = hi[e];
    }
  }
};

// ------------------------------------------------------------------------------------
// y[m][n] = sa[m] sb[n] sum_k a[m][k] b[n][k] + bias[n]
// ------------------------------------------------------------------------------------

struct MatmulArgs {
  const int8_t* a;
  const float* a_scales;
  const int8_t* b;
  const float* b_scales;
  const void* bias;
  int64_t m, n, k;
  void* out;
  int32_t* partial;    // [splits][m][n] where the sum is split
  int splits;
  int steps_per_split;
};

// 16 bytes of a row from byte k on; what lies behind the row's end reads as zero.
__device__ __forceinline__ u32x4 load_bytes(const int8_t* row, int64_t k, int64_t len) {
  if (k + 16 <= len) return *(const u32x4_align1*)(row + k);
  u32x4 v{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (k + i < len) v[i / 4] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i % 4));
  return v;
}

// All bits of the first n of 16 bytes.
__device__ __forceinline__ i32x4 first_bytes(int n) {
  i32x4 v;
#pragma unroll
  for (int w = 0; w < 4; ++w) v[w] = n >= 4 * w + 4 ? -1 : n <= 4 * w ? 0 : (int)((1u << (8 * (n - 4 * w))) - 1u);
  return v;
}

// A tile of R rows of kStep bytes in LDS.  16-byte piece c of row r lies at piece c ^ (r / 2 mod 8).  LDS serves 256
// bytes a cycle, two rows: of the 16 rows that 16 neighbouring lanes read at the same k, the even ones lie in one half of
// the banks and the odd ones in the other, each in eight different places.
constexpr int kStep = 128;
template <int R, int THREADS>
struct ByteTile {
  static constexpr int kPieces = R * (kStep / 16) / THREADS;
  static_assert(R * (kStep / 16) % THREADS == 0, "whole pieces per lane");
  static __device__ __forceinline__ void where(int i, int& row, int& piece) {
    const int p = i * THREADS + threadIdx.x;
    row = p / 8;
    piece = (p % 8) ^ (row / 2 & 7);
  }
  // rows from the buffer's start on, `len` bytes long each, from byte k0 on; a piece behind a row's end is the next row's
  static __device__ __forceinline__ void copy(Buffer src, uint32_t len, uint32_t k0, int8_t* lds) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      int r, c;
      where(i, r, c);
      copy16_to_lds(src, (uint32_t)r * len + k0 + c * 16, lds + (i * THREADS + wave_id() * 64) * 16);
    }
  }
  // the same through registers, for rows that do not start on 16 bytes; rows behind the last are the last one again
  static __device__ __forceinline__ void load(const int8_t* src, int rows, uint32_t len, uint32_t k0, u32x4 (&v)[kPieces]) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      int r, c;
      where(i, r, c);
      v[i] = *(const u32x4_align1*)(src + ((uint32_t)(r < rows ? r : rows - 1) * len + k0 + c * 16));
    }
  }
  static __device__ __forceinline__ void load_last(const int8_t* src, int rows, uint32_t len, uint32_t k0, u32x4 (&v)[kPieces]) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      int r, c;
      where(i, r, c);
      v[i] = r < rows && k0 + c * 16 < len ? load_bytes(src + (uint32_t)r * len, k0 + c * 16, len) : u32x4{0, 0, 0, 0};
    }
  }
  static __device__ __forceinline__ void store(const u32x4 (&v)[kPieces], int8_t* lds) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) *(u32x4*)(lds + (i * THREADS + threadIdx.x) * 16) = v[i];
  }
  // the 16 bytes of row r from piece c on
  static __device__ __forceinline__ i32x4 read(const int8_t* lds, int r, int c) { return *(const i32x4*)(lds + r * kStep + ((c ^ (r / 2 & 7)) * 16)); }
};

// Tiles of BM x BN, WM x WN wavefronts, each with BM/WM x BN/WN of it in registers as 32 x 32 blocks of sums.  The
// weight's rows are the matrix instruction's first operand: a lane then holds four neighbouring channels of a row.
template <int DT, int BM, int BN, int WM, int WN, bool ALIGNED>
__global__ void __launch_bounds__(WM * WN * 64) matmul_kernel(MatmulArgs p) {
  constexpr int kWaves = WM * WN, kThreads = kWaves * 64, kM = BM / WM / 32, kN = BN / WN / 32;
  using TA = ByteTile<BM, kThreads>;
  using TB = ByteTile<BN, kThreads>;
  __shared__ __attribute__((aligned(1024))) int8_t a0[BM * kStep], a1[BM * kStep], b0[BN * kStep], b1[BN * kStep];
  const int tm = (int)((p.m + BM - 1) / BM), tn = (int)((p.n + BN - 1) / BN);
  const int split = blockIdx.x / (tm * tn);
  const Tile tile = tile_of(blockIdx.x % (tm * tn), tm, tn);
  const int64_t m0 = (int64_t)tile.row * BM, n0 = (int64_t)tile.col * BN;
  const int wave = wave_id(), lane = threadIdx.x % 64;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const int all = (int)((p.k + kStep - 1) / kStep);
  const int begin = split * p.steps_per_split, end = begin + p.steps_per_split < all ? begin + p.steps_per_split : all;

  i32x16 acc[kN][kM];
#pragma unroll
  for (int j = 0; j < kN; ++j)
#pragma unroll
    for (int i = 0; i < kM; ++i) acc[j][i] = i32x16{};

  u32x4 va[TA::kPieces], vb[TB::kPieces];
  const Buffer ra = buffer_of(p.a + m0 * p.k, (p.m - m0 < BM ? p.m - m0 : BM) * p.k), rb = buffer_of(p.b + n0 * p.k, (p.n - n0 < BN ? p.n - n0 : BN) * p.k);
  const int8_t *pa = p.a + m0 * p.k, *pb = p.b + n0 * p.k;
  const int rows_a = (int)(p.m - m0 < BM ? p.m - m0 : BM), rows_b = (int)(p.n - n0 < BN ? p.n - n0 : BN);
  const uint32_t len = (uint32_t)p.k;
  auto fetch = [&](int step, auto which) {
    if constexpr (ALIGNED) {
      TA::copy(ra, len, step * kStep, which.value ? a1 : a0);
      TB::copy(rb, len, step * kStep, which.value ? b1 : b0);
    } else {
      TA::load(pa, rows_a, len, step * kStep, va);
      TB::load(pb, rows_b, len, step * kStep, vb);
    }
  };
  auto fetch_last = [&](int step, auto which) {
    if constexpr (ALIGNED) {
      fetch(step, which);
    } else {
      TA::load_last(pa, rows_a, len, step * kStep, va);
      TB::load_last(pb, rows_b, len, step * kStep, vb);
    }
  };
  auto settle = [&](auto which) {
    if constexpr (!ALIGNED) {
      TA::store(va, which.value ? a1 : a0);
      TB::store(vb, which.value ? b1 : b0);
    }
    __syncthreads();
  };
  // `left`: bytes of the sum that are left; what lies behind them in the tiles is not part of it
  const int left = end == all ? (int)(p.k - (int64_t)(all - 1) * kStep) : kStep;
  auto multiply_some = [&](const int8_t* a, const int8_t* b, auto last) {
    i32x4 fa[2][kM], fb[2][kN];
    auto read = [&](int ks, i32x4 (&ra)[kM], i32x4 (&rb)[kN]) {
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        rb[j] = TB::read(b, wn + j * 32 + lane % 32, ks * 2 + lane / 32);
        if (last.value && (ks + 1) * 32 > left) rb[j] &= first_bytes(left - ks * 32 - lane / 32 * 16);
      }
#pragma unroll
      for (int i = 0; i < kM; ++i) ra[i] = TA::read(a, wm + i * 32 + lane % 32, ks * 2 + lane / 32);
    };
    read(0, fa[0], fb[0]);
#pragma unroll
    for (int ks = 0; ks < kStep / 32; ++ks) {  // the next reads are on their way while this slice multiplies
      if (ks + 1 < kStep / 32) read(ks + 1, fa[(ks + 1) % 2], fb[(ks + 1) % 2]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kM; ++i)
#pragma unroll
        for (int j = 0; j < kN; ++j) acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[ks % 2][j], fa[ks % 2][i], acc[j][i], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  run_steps(begin, end, fetch, fetch_last, settle, [&](auto which) { multiply_some(which.value ? a1 : a0, which.value ? b1 : b0, std::false_type{}); },
            [&](auto which) { multiply_some(which.value ? a1 : a0, which.value ? b1 : b0, std::true_type{}); });

  // The sums go through LDS (the second pair of tiles, which nobody reads any more) 32 rows at a time, so that a
  // lane has eight neighbouring channels to scale and to store.
  using E = Elem<DT>;
  using T = typename E::type;
  using O = OutBlock<32, BN / WN>;
  static_assert(kWaves / 2 * O::kBytes <= BM * kStep && kWaves / 2 * O::kBytes <= BN * kStep, "half of the waves' blocks fit either tile");
  uint32_t* block = (uint32_t*)((wave < kWaves / 2 ? a1 : b1) + wave % (kWaves / 2) * O::kBytes);
  const int64_t n = n0 + wn + O::col();
  const int64_t some = p.n - n;
  float sb[8], bias[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    sb[e] = e < some && p.splits == 1 ? p.b_scales[n + e] : 0.0f;
    bias[e] = e < some && p.splits == 1 && p.bias ? E::get(((const T*)p.bias)[n + e]) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < kM; ++i) {
#pragma unroll
    for (int j = 0; j < kN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const u32x4 v{(uint32_t)acc[j][i][q * 4], (uint32_t)acc[j][i][q * 4 + 1], (uint32_t)acc[j][i][q * 4 + 2], (uint32_t)acc[j][i][q * 4 + 3]};
        O::put(block, lane % 32, j * 8 + q * 2 + lane / 32, v);
      }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int t = 0; t < O::kTurns; ++t) {
      const int64_t m = m0 + wm + i * 32 + O::row(t);
      uint32_t v[8];
      O::get(block, O::row(t), v);
      if (m < p.m && some > 0) {
        if (p.splits > 1) {
          store_some<OPTIMI_F32>((float*)p.partial + ((int64_t)split * p.m + m) * p.n + n, reinterpret_cast<const float(&)[8]>(v), some);
        } else {
          const float sa = p.a_scales[m];
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = fmaf((float)(int32_t)v[e] * sa, sb[e], bias[e]);
          store_some<DT>((T*)p.out + m * p.n + n, f, some);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// Adds the splits' whole-number sums, four columns a lane.
template <int DT>
__global__ void __launch_bounds__(256) matmul_finish_kernel(MatmulArgs p) {
  using E = Elem<DT>;
  using T = typename E::type;
  for (int64_t m = blockIdx.y; m < p.m; m += gridDim.y) {
    const int64_t n = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (n >= p.n) continue;
    int32_t sum[4] = {0, 0, 0, 0};
    for (int s = 0; s < p.splits; ++s) {
      const int32_t* from = p.partial + ((int64_t)s * p.m + m) * p.n + n;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.n) sum[e] += from[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (n + e >= p.n) continue;
      const float bias = p.bias ? E::get(((const T*)p.bias)[n + e]) : 0.0f;
      ((T*)p.out)[m * p.n + n + e] = E::put(fmaf((float)sum[e] * p.a_scales[m], p.b_scales[n + e], bias));
    }
  }
}

// ------------------------------------------------------------------------------------
// dw[n][k] = sum_m g[m][n] s[m] q[m][k]
// ------------------------------------------------------------------------------------

struct WeightGradArgs {
  const void* grad;
  const int8_t* values;
  const float* scales;
  int64_t rows, outs, cols;
  void* out;
  float* partial;  // [splits][outs][cols] where the sum is split
  int splits;
  int steps_per_split;
};

template <int DT>
struct Product;
template <>
struct Product<OPTIMI_BF16> {
  static constexpr int kPieces = 1;
  static __device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pair(float a, float b) { return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b}); }
};
template <>
struct Product<OPTIMI_F16> {
  static constexpr int kPieces = 1;
  static __device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pair(float a, float b) { return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b}); }
};
template <>
struct Product<OPTIMI_F32> : Product<OPTIMI_BF16> {
  static constexpr int kPieces = 3;
};

// The upper 8 bits of two fp32 numbers as two bf16 ones; what is left of them stays in x.  Three times over, the
// pieces add up to the number exactly.  Numbers that are not finite leave nothing.
__device__ __forceinline__ uint32_t split_pair(float& x, float& y) {
  const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
  const bool fx = abs_bits(x) < 0x7f800000u, fy = abs_bits(y) < 0x7f800000u;
  x = fx ? x - __uint_as_float(a & 0xffff0000u) : 0.0f;
  y = fy ? y - __uint_as_float(b & 0xffff0000u) : 0.0f;
  // a NaN whose upper half would be an infinity's becomes a quiet one
  const uint32_t ha = a | ((a & 0x7fffffffu) > 0x7f800000u ? 0x400000u : 0u), hb = b | ((b & 0x7fffffffu) > 0x7f800000u ? 0x400000u : 0u);
  return __builtin_amdgcn_perm(hb, ha, 0x07060302u);
}

// The sum runs over rows, and both operands lie in memory with their rows' columns side by side, so the matrix
// instruction wants both of them transposed.  Tiles go to LDS as they are, [rows][columns] of 16 bits, and gfx950's
// transposing LDS read takes a 16-row column out of them: four rows x 16 columns per 16 lanes.  In one such read
// a wave touches 16 rows; 32-byte chunk c of row r lies at chunk c ^ (r mod the chunks of a row), which spreads them over the banks.
template <int C>
struct HalfTile {
  static constexpr int kChunks = C / 16;
  static __device__ __forceinline__ int at(int row, int chunk) { return row * C + ((chunk ^ (row & (kChunks - 1) & 15)) * 16); }  // in elements
};

template <int DT, int BN, int BC, int WN, int WC, int STEP, bool DIRECT, bool NARROW = false>
__global__ void __launch_bounds__(WN * WC * 64) weight_grad_kernel(WeightGradArgs p) {
  using E = Elem<DT>;
  using T = typename E::type;
  using P = Product<DT>;
  constexpr int kWaves = WN * WC, kThreads = kWaves * 64, kN = BN / WN / 16, kC = BC / WC / 16;
  constexpr int kPieces = P::kPieces;
  using TG = HalfTile<BN>;
  using TQ = HalfTile<BC>;
  __shared__ __attribute__((aligned(1024))) short g0[kPieces * STEP * BN], g1[kPieces * STEP * BN], q0[STEP * BC], q1[STEP * BC];
  const int tn = (int)((p.outs + BN - 1) / BN), tc = (int)((p.cols + BC - 1) / BC);
  const int split = blockIdx.x / (tn * tc);
  const Tile tile = tile_of(blockIdx.x % (tn * tc), tn, tc);
  const int64_t n0 = (int64_t)tile.row * BN, c0 = (int64_t)tile.col * BC;
  const int wave = wave_id(), lane = threadIdx.x % 64;
  const int wn = wave / WC * (BN / WN), wc = wave % WC * (BC / WC);
  const int all = (int)((p.rows + STEP - 1) / STEP);
  const int begin = split * p.steps_per_split, end = begin + p.steps_per_split < all ? begin + p.steps_per_split : all;

  f32x4 acc[kN][kC];
#pragma unroll
  for (int i = 0; i < kN; ++i)
#pragma unroll
    for (int j = 0; j < kC; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  // per lane: kGrad pieces of 8 gradients, kQ pieces of 16 values
  constexpr int kGrad = STEP * BN / 8 / kThreads, kQ = STEP * BC / 16 / kThreads;
  static_assert(kGrad * 8 * kThreads == STEP * BN && kQ * 16 * kThreads == STEP * BC, "whole pieces per lane");
  typename E::Raw vg[kGrad];
  float sg[kGrad];
  u32x4 vq[kQ];
  float sq[kQ];
  const int outs = (int)(p.outs - n0 < BN ? p.outs - n0 : BN), cols = (int)(p.cols - c0 < BC ? p.cols - c0 : BC);
  auto copy = [&](int64_t m0, int rows, short* g) {  // LDS place -> row, place in row; the source follows the swizzle
    const Buffer from = buffer_of((const T*)p.grad + m0 * p.outs + n0, ((int64_t)(rows - 1) * p.outs + outs) * 2);
#pragma unroll
    for (int i = 0; i < kGrad; ++i) {
      const int place = i * kThreads + threadIdx.x;
      const int row = place / (BN / 8), in = place % (BN / 8);
      const int n = TG::at(row, in / 2) - row * BN + in % 2 * 8;
      copy16_to_lds(from, ((uint32_t)row * (uint32_t)p.outs + n) * 2, g + (i * kThreads + wave * 64) * 8);
    }
  };
  // A full step's loads.  Columns behind the matrix are read from its first ones and never used; a piece that begins inside
  // may run into the next row, of which there is one.
  auto fetch = [&](int step, auto which) {
    const int64_t m0 = (int64_t)step * STEP;
    const T* grad = (const T*)p.grad + m0 * p.outs + n0;
    const int8_t* values = p.values + m0 * p.cols + c0;
    const float* scales = p.scales + m0;
    if constexpr (DIRECT) {
      copy(m0, STEP, which.value ? g1 : g0);
    } else {
#pragma unroll
      for (int i = 0; i < kGrad; ++i) {
        const int place = i * kThreads + threadIdx.x;
        const int row = place / (BN / 8), n = place % (BN / 8) * 8;
        vg[i] = E::load(grad + ((uint32_t)row * (uint32_t)p.outs + (n < outs ? n : 0)));
        if (kPieces > 1) sg[i] = scales[row];
      }
    }
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      const int place = i * kThreads + threadIdx.x;
      const int row = place / (BC / 16), c = place % (BC / 16) * 16;
      vq[i] = *(const u32x4_align1*)(values + ((uint32_t)row * (uint32_t)p.cols + (c < cols ? c : 0)));
      sq[i] = kPieces > 1 ? 1.0f : scales[row];
    }
  };
  // The last step's, or any step's of a matrix that is narrower than a piece.
  auto fetch_last = [&](int step, auto which) {
    const int64_t m0 = (int64_t)step * STEP;
    const T* grad = (const T*)p.grad + m0 * p.outs + n0;
    const int8_t* values = p.values + m0 * p.cols + c0;
    const float* scales = p.scales + m0;
    const int rows = (int)(p.rows - m0 < STEP ? p.rows - m0 : STEP);
    if constexpr (DIRECT) {
      copy(m0, rows, which.value ? g1 : g0);
    } else {
#pragma unroll
      for (int i = 0; i < kGrad; ++i) {
        const int place = i * kThreads + threadIdx.x;
        const int row = place / (BN / 8), n = place % (BN / 8) * 8;
        const bool in = row < rows && n < outs;
        vg[i] = in ? load_some<DT>(grad + (uint32_t)row * (uint32_t)p.outs + n, outs - n) : E::zero();
        if (kPieces > 1) sg[i] = in ? scales[row] : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      const int place = i * kThreads + threadIdx.x;
      const int row = place / (BC / 16), c = place % (BC / 16) * 16;
      const bool in = row < rows && c < cols;
      vq[i] = in ? load_bytes(values + (uint32_t)row * (uint32_t)p.cols, c, cols) : u32x4{0, 0, 0, 0};
      sq[i] = kPieces > 1 ? 1.0f : in ? scales[row] : 0.0f;
    }
  };
  auto settle = [&](auto which) {
    short *g = which.value ? g1 : g0, *q = which.value ? q1 : q0;
    if constexpr (!DIRECT) {
#pragma unroll
      for (int i = 0; i < kGrad; ++i) {
        const int place = i * kThreads + threadIdx.x;
        const int row = place / (BN / 8), in = place % (BN / 8);
        short* to = g + TG::at(row, in / 2) + in % 2 * 8;
        if constexpr (kPieces == 1) {
          *(u32x4*)to = vg[i].a;
        } else {
          float f[8];
          E::unpack(vg[i], f);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= sg[i];
#pragma unroll
          for (int z = 0; z < kPieces; ++z) {
            u32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = split_pair(f[2 * e], f[2 * e + 1]);
            *(u32x4*)(to + z * STEP * BN) = v;
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      const int place = i * kThreads + threadIdx.x;
      short* to = q + TQ::at(place / (BC / 16), place % (BC / 16));
      const float s = sq[i], minus = -128.0f * s;
      u32x4 v[2];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        // bytes as unsigned numbers, 128 too large: (u - 128) s with one rounding
        const uint32_t u = vq[i][w] ^ 0x80808080u;
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = fmaf((float)((u >> (8 * e)) & 0xffu), s, minus);
        v[w / 2][w % 2 * 2] = P::pair(f[0], f[1]);
        v[w / 2][w % 2 * 2 + 1] = P::pair(f[2], f[3]);
      }
      *(u32x4*)to = v[0];
      *(u32x4*)(to + 8) = v[1];
    }
    __syncthreads();
  };
  // rows 32 ks .. 32 ks + 31 of 16 columns, as the matrix instruction takes them (in an order of rows that is the same for both operands)
  auto column = [&](const short* t, int pitch, int offset, int ks) {
    typedef OPTIMI_LDS s16x4* Ptr;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(t + offset + ks * 32 * pitch));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(t + offset + (ks * 32 + 16) * pitch));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // `left`: rows of the sum that are left.  The values behind them are zeros, but a copied gradient tile holds
  // whatever was in LDS there, infinities maybe.
  const int left = end == all ? (int)(p.rows - (int64_t)(all - 1) * STEP) : STEP;
  auto multiply_some = [&](const short* g, const short* q, auto last) {
#pragma unroll
    for (int ks = 0; ks < STEP / 32; ++ks) {
      s16x8 fq[kC], keep;
      if (last.value) {
#pragma unroll
        for (int e = 0; e < 8; ++e) keep[e] = ks * 32 + e / 4 * 16 + lane / 16 * 4 + e % 4 < left ? -1 : 0;
      }
#pragma unroll
      for (int j = 0; j < kC; ++j) fq[j] = column(q, BC, TQ::at(lane / 4, wc / 16 + j) + lane % 4 * 4, ks);
#pragma unroll
      for (int z = kPieces - 1; z >= 0; --z)
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          s16x8 fg = column(g + z * STEP * BN, BN, TG::at(lane / 4, wn / 16 + i) + lane % 4 * 4, ks);
          if (last.value) fg &= keep;
#pragma unroll
          for (int j = 0; j < kC; ++j) acc[i][j] = P::mfma(fq[j], fg, acc[i][j]);
        }
    }
  };

  auto fetch_any = [&](int step, auto which) {
    if constexpr (NARROW) fetch_last(step, which);
    else fetch(step, which);
  };
  run_steps(begin, end, fetch_any, fetch_last, settle, [&](auto which) { multiply_some(which.value ? g1 : g0, which.value ? q1 : q0, std::false_type{}); },
            [&](auto which) { multiply_some(which.value ? g1 : g0, which.value ? q1 : q0, std::bool_constant<DIRECT>{}); });

  using O = OutBlock<16, BC / WC>;
  static_assert(kWaves / 2 * O::kBytes <= STEP * BC * 2 && kWaves / 2 * O::kBytes <= STEP * BN * 2, "half of the waves' blocks fit either tile");
  uint32_t* block = (uint32_t*)((char*)(wave < kWaves / 2 ? g1 : q1) + wave % (kWaves / 2) * O::kBytes);
  const int64_t c = c0 + wc + O::col();
  const int64_t some = p.cols - c;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
#pragma unroll
    for (int j = 0; j < kC; ++j) O::put(block, lane % 16, j * 4 + lane / 16, __builtin_bit_cast(u32x4, acc[i][j]));
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int t = 0; t < O::kTurns; ++t) {
      const int64_t n = n0 + wn + i * 16 + O::row(t);
      uint32_t v[8];
      O::get(block, O::row(t), v);
      const float(&f)[8] = reinterpret_cast<const float(&)[8]>(v);
      if (n < p.outs && some > 0) {
        if (p.splits > 1) store_some<OPTIMI_F32>(p.partial + ((int64_t)split * p.outs + n) * p.cols + c, f, some);
        else store_some<DT>((T*)p.out + n * p.cols + c, f, some);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The same for large 16-bit products, where all that counts is that the matrix instructions never wait: 256 x 256 tiles, 64
// rows a step, two pairs of tiles in LDS, eight wavefronts with 128 x 64 sums each.  Gradients go to LDS past the registers;
// the values have to become 16-bit numbers on the way, and are loaded two steps ahead, so that the conversion of the next
// step's values can be spread over this step's products without waiting for memory.  outs is a multiple of 8, grad aligned to
// 16 bytes, and there are 16 values at least.
template <int DT>
__global__ void __launch_bounds__(512) weight_grad_wide_kernel(WeightGradArgs p) {
  using T = typename Elem<DT>::type;
  using P = Product<DT>;
  constexpr int kTile = 256, kRows = 64, kN = 8, kC = 4, kPieces = 2;
  using H = HalfTile<kTile>;
  __shared__ __attribute__((aligned(1024))) short g0[kRows * kTile], g1[kRows * kTile], q0[kRows * kTile], q1[kRows * kTile];
  const int tn = (int)((p.outs + kTile - 1) / kTile), tc = (int)((p.cols + kTile - 1) / kTile);
  const int split = blockIdx.x / (tn * tc);
  const Tile tile = tile_of(blockIdx.x % (tn * tc), tn, tc);
  const int64_t n0 = (int64_t)tile.row * kTile, c0 = (int64_t)tile.col * kTile;
  const int wave = wave_id(), lane = threadIdx.x % 64;
  const int wn = wave / 4 * 128, wc = wave % 4 * 64;
  const int all = (int)((p.rows + kRows - 1) / kRows);
  const int begin = split * p.steps_per_split, end = begin + p.steps_per_split < all ? begin + p.steps_per_split : all;

  f32x4 acc[kN][kC];
#pragma unroll
  for (int i = 0; i < kN; ++i)
#pragma unroll
    for (int j = 0; j < kC; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  // Gradients: a wave's copy fills two rows of LDS; the sources follow the swizzle.  Columns behind the matrix come from the
  // next row (or not at all, behind the last) and end in sums that are not stored.
  const int outs = (int)(p.outs - n0 < kTile ? p.outs - n0 : kTile);
  auto copy = [&](int step, short* g) {
    const int64_t m0 = (int64_t)step * kRows;
    const int rows = (int)(p.rows - m0 < kRows ? p.rows - m0 : kRows);
    const Buffer from = buffer_of((const T*)p.grad + m0 * p.outs + n0, ((int64_t)(rows - 1) * p.outs + outs) * 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int place = i * 512 + threadIdx.x;
      const int row = place / 32, in = place % 32;
      const int n = H::at(row, in / 2) - row * kTile + in % 2 * 8;
      copy16_to_lds(from, ((uint32_t)row * (uint32_t)p.outs + n) * 2, g + (i * 512 + wave * 64) * 8);
    }
  };
  // Values: a lane has 16 neighbours of two rows.  Rows behind the last are the last one again, under a scale of 0;
  // columns behind the matrix are never used.  A piece that would run over the end of all values is loaded from a little
  // before, and shifted into its place when it is converted.
  const int64_t total = p.rows * p.cols;
  const int at_row = threadIdx.x / 16, at_col = threadIdx.x % 16;
  const uint32_t col = (uint32_t)c0 + (c0 + at_col * 16 < p.cols ? at_col * 16 : 0);
  u32x4 vq[2][kPieces];
  float sq[2][kPieces];
  auto place_of = [&](int step, int i, int64_t& start, uint32_t& limit) {
    const int64_t m0 = (int64_t)step * kRows, first = m0 * p.cols;
    start = first < total - 16 ? first : total - 16;
    const int64_t left = total - 16 - start;
    limit = (uint32_t)(left < 0x7fffffff ? left : 0x7fffffff);
    const int rows = (int)(p.rows - m0 < kRows ? p.rows - m0 : kRows), row = at_row + i * 32;
    return (uint32_t)(row < rows ? row : rows - 1) * (uint32_t)p.cols + col + (uint32_t)(first - start);
  };
  auto load = [&](int step, u32x4 (&v)[kPieces], float (&s)[kPieces]) {
    const int64_t m0 = (int64_t)step * kRows;
    const int rows = (int)(p.rows - m0 < kRows ? p.rows - m0 : kRows);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      int64_t start;
      uint32_t limit;
      const uint32_t at = place_of(step, i, start, limit);
      v[i] = *(const u32x4_align1*)(p.values + start + (at < limit ? at : limit));
      const int row = at_row + i * 32;
      s[i] = p.scales[m0 + (row < rows ? row : rows - 1)];
    }
  };
  auto shift = [&](int step, u32x4 (&v)[kPieces], float (&s)[kPieces]) {  // the very last step only
    const int rows = (int)(p.rows - (int64_t)step * kRows);
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      int64_t start;
      uint32_t limit;
      const uint32_t at = place_of(step, i, start, limit), by = at > limit ? (at - limit) * 8 : 0;
      uint64_t lo = (uint64_t)v[i][1] << 32 | v[i][0], hi = (uint64_t)v[i][3] << 32 | v[i][2];
      if (by >= 64) {
        lo = hi >> (by - 64 & 63);
        hi = 0;
      } else if (by > 0) {
        lo = lo >> by | hi << (64 - by);
        hi >>= by;
      }
      v[i] = u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
      if (at_row + i * 32 >= rows) s[i] = 0.0f;
    }
  };
  // Four values as 16-bit numbers: bytes as unsigned numbers are 128 too large, (u - 128) s has one rounding, and none
  // under a power of two.
  auto convert = [&](uint32_t word, float s) {
    const uint32_t u = word ^ 0x80808080u;
    const float minus = -128.0f * s;
    float f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = fmaf((float)((u >> (8 * e)) & 0xffu), s, minus);
    return u32x2{P::pair(f[0], f[1]), P::pair(f[2], f[3])};
  };
  auto write_half = [&](int half, const u32x4 (&v)[kPieces], const float (&s)[kPieces], short* q) {  // eight values of piece half / 2
    const int i = half / 2;
    const u32x2 a = convert(v[i][half % 2 * 2], s[i]), b = convert(v[i][half % 2 * 2 + 1], s[i]);
    *(u32x4*)(q + H::at(at_row + i * 32, at_col) + half % 2 * 8) = u32x4{a[0], a[1], b[0], b[1]};
  };

  // Where a lane's part of 16 columns lies: chunks differ in five address bits only, so chunk i of the wave's is one
  // exclusive or away from its first.  The addresses are formed anew for every step: kept over the loop, they would take more
  // registers than there are.
  typedef OPTIMI_LDS s16x4* Ptr;
  auto column = [&](const short* t, int first, int i, int ks) {
    const char* from = (const char*)t + (first ^ (i * 32)) + ks * 32 * kTile * 2;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)from);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(from + 16 * kTile * 2));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto anew = [](int v) {
    asm volatile("" : "+v"(v));
    return v & 0x7fff;
  };
  const int first_g = (H::at(lane / 4, wn / 16) + lane % 4 * 4) * 2, first_q = (H::at(lane / 4, wc / 16) + lane % 4 * 4) * 2;
  const int left = end == all ? (int)(p.rows - (int64_t)(all - 1) * kRows) : kRows;
  // One step's products in sixteen groups; a group's operands are read two groups earlier, and four of the groups are followed
  // by a quarter of the next step's conversion.
  auto multiply = [&](const short* g, const short* q, auto last, const u32x4 (&v)[kPieces], const float (&s)[kPieces], short* next) {
    const int at_g = anew(first_g), at_q = anew(first_q);
    s16x8 fq[2][kC], fg[3];
    auto keep = [&](s16x8 f, int ks) {  // copied gradients of rows behind the last are whatever was in LDS, infinities maybe
      if (!last.value) return f;
      s16x8 mask;
#pragma unroll
      for (int e = 0; e < 8; ++e) mask[e] = ks * 32 + e / 4 * 16 + lane / 16 * 4 + e % 4 < left ? -1 : 0;
      return f & mask;
    };
#pragma unroll
    for (int j = 0; j < kC; ++j) fq[0][j] = column(q, at_q, j, 0);
    fg[0] = column(g, at_g, 0, 0);
    fg[1] = column(g, at_g, 1, 0);
#pragma unroll
    for (int t = 0; t < 2 * kN; ++t) {
      const int ks = t / kN, i = t % kN;
      if (t + 2 < 2 * kN) fg[(t + 2) % 3] = column(g, at_g, (t + 2) % kN, (t + 2) / kN);
      if (t == 3) {
#pragma unroll
        for (int j = 0; j < kC; ++j) fq[1][j] = column(q, at_q, j, 1);
      }
      const s16x8 f = keep(fg[t % 3], ks);
#pragma unroll
      for (int j = 0; j < kC; ++j) acc[i][j] = P::mfma(fq[ks][j], f, acc[i][j]);
      if (!last.value && t % 3 == 1 && t / 3 < 2 * kPieces) write_half(t / 3, v, s, next);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto step_on = [&](int step, auto which) {
    constexpr int W = decltype(which)::value;
    copy(step + 1, W ? g0 : g1);
    if (step + 2 < end) load(step + 2, vq[W], sq[W]);
    if (step + 2 == all) shift(step + 1, vq[1 - W], sq[1 - W]);
    __builtin_amdgcn_sched_barrier(0);  // the loads start before the products do; left alone, they are moved behind them
    multiply(W ? g1 : g0, W ? q1 : q0, std::false_type{}, vq[1 - W], sq[1 - W], W ? q0 : q1);
    __syncthreads();
  };
  auto start = [&](int step, auto which) {
    constexpr int W = decltype(which)::value;
    copy(step, W ? g1 : g0);
    load(step, vq[W], sq[W]);
    if (step + 1 < end) load(step + 1, vq[1 - W], sq[1 - W]);
    if (step + 1 == all) shift(step, vq[W], sq[W]);
#pragma unroll
    for (int half = 0; half < 2 * kPieces; ++half) write_half(half, vq[W], sq[W], W ? q1 : q0);
    __syncthreads();
  };

  // the last step works on the first pair of tiles
  if (begin < end) {
    int step = begin;
    if ((end - begin) % 2) {
      start(step, Pair<0>{});
    } else {
      start(step, Pair<1>{});
      step_on(step++, Pair<1>{});
    }
    for (; step + 1 < end; step += 2) {
      step_on(step, Pair<0>{});
      step_on(step + 1, Pair<1>{});
    }
    multiply(g0, q0, std::true_type{}, vq[0], sq[0], q1);
  }

  using O = OutBlock<16, 64>;
  uint32_t* block = (uint32_t*)((char*)(wave < 4 ? g1 : q1) + wave % 4 * O::kBytes);
  const int64_t c = c0 + wc + O::col();
  const int64_t some = p.cols - c;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
#pragma unroll
    for (int j = 0; j < kC; ++j) O::put(block, lane % 16, j * 4 + lane / 16, __builtin_bit_cast(u32x4, acc[i][j]));
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int t = 0; t < O::kTurns; ++t) {
      const int64_t n = n0 + wn + i * 16 + O::row(t);
      uint32_t v[8];
      O::get(block, O::row(t), v);
      const float(&f)[8] = reinterpret_cast<const float(&)[8]>(v);
      if (n < p.outs && some > 0) {
        if (p.splits > 1) store_some<OPTIMI_F32>(p.partial + ((int64_t)split * p.outs + n) * p.cols + c, f, some);
        else store_some<DT>((T*)p.out + n * p.cols + c, f, some);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// Adds the splits' sums, always in the same order.
template <int DT>
__global__ void __launch_bounds__(256) weight_grad_finish_kernel(WeightGradArgs p) {
  using E = Elem<DT>;
  const int64_t n = p.outs * p.cols;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (i + e >= n) break;
      float sum = 0.0f;
      for (int s = 0; s < p.splits; ++s) sum += p.partial[s * n + i + e];
      ((typename E::type*)p.out)[i + e] = E::put(sum);
    }
  }
}

template <class F>
int by_dtype(int dtype, F f) {
  switch (dtype) {
    case OPTIMI_F32: return f(std::integral_constant<int, OPTIMI_F32>{});
    case OPTIMI_BF16: return f(std::integral_constant<int, OPTIMI_BF16>{});
    default: return f(std::integral_constant<int, OPTIMI_F16>{});
  }
}

constexpr int64_t kMostWidth = 1 << 24;  // of a weight gradient: offsets inside a tile stay in 31 bits
constexpr int64_t kMostSum = 131071;  // (-128)^2 times this stays below 2^31
constexpr int64_t kMostTiles = 1 << 22;  // workgroups of a launch, at most 512 lanes each

// How a product is cut: the tile's size and the number of parts that the sum is split into.
struct Cut {
  int tile;
  int64_t tiles;
  int splits, steps_per_split;
};
constexpr int kCus = 256;
Cut cut(int64_t rows, int64_t cols, int64_t steps, int large, int small) {
  Cut c;
  auto tiles = [&](int t) { return ((rows + t - 1) / t) * ((cols + t - 1) / t); };
  c.tile = tiles(large) >= kCus / 2 ? large : small;
  c.tiles = tiles(c.tile);
  c.splits = 1;
  if (c.tiles < kCus) {
    int64_t s = kCus / c.tiles;
    if (s > steps / 4) s = steps / 4;
    if (s > 16) s = 16;
    if (s > 1) c.splits = (int)s;
  }
  c.steps_per_split = (int)((steps + c.splits - 1) / c.splits);
  if (c.splits > 1) c.splits = (int)((steps + c.steps_per_split - 1) / c.steps_per_split);
  return c;
}
Cut matmul_cut(int64_t m, int64_t n, int64_t k) { return cut(m, n, (k + kStep - 1) / kStep, 256, 64); }
Cut weight_grad_cut(int64_t rows, int64_t outs, int64_t cols, int dtype) {
  return dtype == OPTIMI_F32 || outs < 8 || cols < 16 ? cut(outs, cols, (rows + 31) / 32, 128, 128) : cut(outs, cols, (rows + 63) / 64, 256, 128);
}

}  // namespace

extern "C" {

int64_t optimi_hip_int8_matmul_workspace(int64_t m, int64_t n, int64_t k) {
  if (int rc = check_shape(m, n)) return rc;
  if (k < 0 || k > kMostSum) return OPTIMI_ERR_SIZE;
  if (m == 0 || n == 0) return 0;
  const Cut c = matmul_cut(m, n, k);
  return c.splits > 1 ? c.splits * m * n * 4 : 0;
}

int optimi_hip_int8_matmul(const int8_t* a, const float* a_scales, const int8_t* b, const float* b_scales, const void* bias, int64_t m, int64_t n,
                           int64_t k, int dtype, void* out, void* workspace, optimi_stream_t stream_) {
  if (!valid_dtype(dtype)) return OPTIMI_ERR_DTYPE;
  if (int rc = check_shape(m, n)) return rc;
  if (k < 0 || k > kMostSum) return OPTIMI_ERR_SIZE;
  if (m == 0 || n == 0) return 0;
  if (!a_scales || !b_scales || !out || (k && (!a || !b))) return OPTIMI_ERR_NULL;
  const int64_t size = elem_bytes(dtype);
  if (!aligned_to(a_scales, 4) || !aligned_to(b_scales, 4) || !aligned_to(bias, size) || !aligned_to(out, size) || !aligned_to(workspace, 4)) return OPTIMI_ERR_ALIGN;
  const Cut c = matmul_cut(m, n, k);
  if (c.tiles * c.splits > kMostTiles) return OPTIMI_ERR_SIZE;
  if (c.splits > 1 && !workspace) return OPTIMI_ERR_NULL;
  hipStream_t stream = (hipStream_t)stream_;
  const MatmulArgs args{a, a_scales, b, b_scales, bias, m, n, k, out, (int32_t*)workspace, c.splits, c.steps_per_split};
  const bool aligned = k % 16 == 0 && aligned_to(a, 16) && aligned_to(b, 16);
  return by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const dim3 grid((unsigned)(c.tiles * c.splits));
    if (c.tile == 256) {
      if (aligned) matmul_kernel<DT, 256, 256, 2, 4, true><<<grid, dim3(512), 0, stream>>>(args);
      else matmul_kernel<DT, 256, 256, 2, 4, false><<<grid, dim3(512), 0, stream>>>(args);
    } else {
      if (aligned) matmul_kernel<DT, 64, 64, 2, 2, true><<<grid, dim3(256), 0, stream>>>(args);
      else matmul_kernel<DT, 64, 64, 2, 2, false><<<grid, dim3(256), 0, stream>>>(args);
    }
    OPTIMI_INT8_TRY(hipGetLastError());
    if (c.splits > 1) {
      matmul_finish_kernel<DT><<<dim3((unsigned)((n + 1023) / 1024), (unsigned)(m < 65535 ? m : 65535)), dim3(256), 0, stream>>>(args);
      OPTIMI_INT8_TRY(hipGetLastError());
    }
    return 0;
  });
}

// The workspace: partial sums of the split product, then those of the bias gradient.
int64_t optimi_hip_int8_weight_grad_workspace(int64_t rows, int64_t outs, int64_t cols, int dtype, int with_bias) {
  if (!valid_dtype(dtype)) return OPTIMI_ERR_DTYPE;
  if (int rc = check_shape(rows, outs)) return rc;
  if (int rc = check_shape(rows, cols)) return rc;
  if (outs > kMostWidth || cols > kMostWidth) return OPTIMI_ERR_SIZE;
  if (outs == 0) return 0;
  const Cut c = cols ? weight_grad_cut(rows, outs, cols, dtype) : Cut{1, 1, 1, 0};
  return (c.splits > 1 ? c.splits * outs * cols * 4 : 0) + (with_bias ? column_sum_workspace(rows, outs) : 0);
}

int optimi_hip_int8_weight_grad(const void* grad, const int8_t* values, const float* scales, int64_t rows, int64_t outs, int64_t cols, int dtype,
                                void* weight_grad, void* bias_grad, void* workspace, optimi_stream_t stream_) {
  if (!valid_dtype(dtype)) return OPTIMI_ERR_DTYPE;
  if (int rc = check_shape(rows, outs)) return rc;
  if (int rc = check_shape(rows, cols)) return rc;
  if (outs > kMostWidth || cols > kMostWidth) return OPTIMI_ERR_SIZE;
  if (outs == 0) return 0;
  if ((cols && !weight_grad) || (rows && (!grad || !scales || (cols && !values))) || (rows && bias_grad && !workspace)) return OPTIMI_ERR_NULL;
  const int64_t size = elem_bytes(dtype);
  if (!aligned_to(grad, size) || !aligned_to(scales, 4) || !aligned_to(weight_grad, size) || !aligned_to(bias_grad, size) || !aligned_to(workspace, 4))
    return OPTIMI_ERR_ALIGN;
  hipStream_t stream = (hipStream_t)stream_;
  const Cut c = cols ? weight_grad_cut(rows, outs, cols, dtype) : Cut{1, 1, 1, 0};
  if (c.tiles * c.splits > kMostTiles) return OPTIMI_ERR_SIZE;
  if (c.splits > 1 && !workspace) return OPTIMI_ERR_NULL;
  if (bias_grad) {
    float* sums = (float*)workspace + (c.splits > 1 ? c.splits * outs * cols : 0);
    if (int rc = column_sum(grad, rows, outs, dtype, bias_grad, sums, stream)) return rc;
  }
  if (cols == 0) return 0;
  const WeightGradArgs args{grad, values, scales, rows, outs, cols, weight_grad, (float*)workspace, c.splits, c.steps_per_split};
  return by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const dim3 grid((unsigned)(c.tiles * c.splits));
    if (outs < 8 || cols < 16) {  // too narrow for whole pieces: every step looks at the borders
      weight_grad_kernel<DT, 128, 128, 2, 2, 32, false, true><<<grid, dim3(256), 0, stream>>>(args);
    } else if constexpr (DT == OPTIMI_F32) {
      weight_grad_kernel<DT, 128, 128, 2, 2, 32, false><<<grid, dim3(256), 0, stream>>>(args);
    } else {
      const bool direct = outs % 8 == 0 && aligned_to(grad, 16);
      if (c.tile == 256) {
        if (direct) weight_grad_wide_kernel<DT><<<grid, dim3(512), 0, stream>>>(args);
        else weight_grad_kernel<DT, 256, 256, 2, 4, 64, false><<<grid, dim3(512), 0, stream>>>(args);
      } else {
        if (direct) weight_grad_kernel<DT, 128, 128, 2, 2, 64, true><<<grid, dim3(256), 0, stream>>>(args);
        else weight_grad_kernel<DT, 128, 128, 2, 2, 64, false><<<grid, dim3(256), 0, stream>>>(args);
      }
    }
    OPTIMI_INT8_TRY(hipGetLastError());
    if (c.splits > 1) {
      const int64_t blocks = (outs * cols + 1023) / 1024;
      weight_grad_finish_kernel<DT><<<dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, stream>>>(args);
      OPTIMI_INT8_TRY(hipGetLastError());
    }
    return 0;
  });
}

}  // extern "C"
