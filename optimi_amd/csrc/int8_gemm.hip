// Matrix products of the int8 activations for MI355X (gfx950): the int8 product with scales per row and channel,
// and the weight gradient taken from an int8 checkpoint.
//
//   y[m][n]  = sa[m] sb[n] sum_k a[m][k] b[n][k] + bias[n]     whole numbers: exact sums in 32 bits, scaled at the end
//   dw[n][k] = sum_m g[m][n] (s[m] q[m][k])                    a scale per term of the sum: it has to go into an operand
//
// The first takes the int8 matrix instructions.  The second takes the 16-bit ones: s q is a whole number below 128 times a
// power of two, which bf16 holds exactly, so the values are widened on their way to LDS and the only roundings left are those of
// the fp32 sums.  (fp16 holds it too, but for values below its subnormal numbers.)  fp32 gradients are cut into three bf16
// pieces, which hold them exactly, and cost three products.
//
// Large products are bound by the matrix instructions and by the power that they draw (the clock falls to 2.0 GHz under them),
// middle ones by how fast a step's tiles get to LDS, those of a few rows by reading the weight, and small ones by the launch.
// Each regime has a kernel; which one is chosen by a cost in measured time per step (matmul_cut, weight_grad_cut).

#include "int8_common.h"

namespace {

using namespace optimi_int8;

typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// The kernels' steps are written as lambdas over their sums and tiles; one that is called instead of inlined would send all
// of them through memory.
#define OPTIMI_INLINE __attribute__((always_inline))
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

// All of this wave's copies and loads are done, and everybody's are: said outright, since a copy to LDS is an access to
// memory that a barrier by itself does not wait for.
__device__ __forceinline__ void meet() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64); }

// Consecutive workgroups go to the eight XCDs in turn, and each XCD has an L2 of its own.  An XCD gets a contiguous
// run of tiles instead, and runs walk the tiles in stripes of kStripe tile rows, so that the tiles in work on
// one XCD at a time form a patch that shares its operands' rows in L2.  (Int8 product 8192 x 11008 x 4096 with stripes of 2, 4,
// 8 and 16: 362, 343, 364, 364 us; weight gradient of these sizes: 766, 737, 746, 745 us.)
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

// The steps [begin, end) of a sum over two pairs of tiles in LDS, copied there asynchronously: while one pair is multiplied, the
// next step's copies are on their way.  fetch(step, which) starts them, multiply(which, last) adds a pair's products;
// the last step works on the first pair, so that the second is free when the sums are done.
template <int I>
using Pair = std::integral_constant<int, I>;
template <class Fetch, class Multiply>
__device__ __forceinline__ void run_copied(int begin, int end, Fetch fetch, Multiply multiply) {
  const Pair<0> p0;
  const Pair<1> p1;
  const std::false_type more;
  if (begin >= end) return;
  int step = begin;
  if ((end - begin) % 2) {
    fetch(step, p0);
    meet();
  } else {
    fetch(step, p1);
    meet();
    fetch(++step, p0);
    __builtin_amdgcn_sched_barrier(0);  // the copies start before the products do; left alone, they are moved behind them
    multiply(p1, more);
    meet();
  }
  for (; step + 1 < end; step += 2) {
    fetch(step + 1, p1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(p0, more);
    meet();
    fetch(step + 2, p0);
    __builtin_amdgcn_sched_barrier(0);
    multiply(p1, more);
    meet();
  }
  multiply(p0, std::true_type{});
}

// The same through registers, which can be loaded from any address: load(step, part, last) starts the loads of a step that is two
// ahead, write(which, part) brings a part that has arrived to LDS, multiply(which, more, part) adds a pair's products
// and, with `more`, does what write() does to the other pair on the way.  Only the last step's loads look at the matrices'
// borders, and they are not told apart inside the loop: a branch around loads makes the compiler wait for all of them in
// front of the next ones.
template <class Part, class Load, class Write, class Multiply>
__device__ __forceinline__ void run_loaded(int begin, int end, Part (&part)[2], Load load, Write write, Multiply multiply) {
  const Pair<0> p0;
  const Pair<1> p1;
  const std::false_type ordinary, no_more;
  const std::true_type last, more;
  auto loaded_step = [&](int step, auto which, auto is_last) OPTIMI_INLINE {
    constexpr int W = decltype(which)::value;
    load(step + 2, part[W], is_last);
    __builtin_amdgcn_sched_barrier(0);
    multiply(which, more, part[1 - W]);
    __syncthreads();
  };
  const int n = end - begin;
  if (n <= 0) return;
  if (n == 1) {
    load(begin, part[0], last);
    write(p0, part[0]);
    __syncthreads();
  } else {
    if (n == 2) {
      load(begin, part[1], ordinary);
      load(begin + 1, part[0], last);
      write(p1, part[1]);
      __syncthreads();
    } else {
      int step = begin;
      if (n % 2) {
        load(step, part[0], ordinary);
        load(step + 1, part[1], ordinary);
        write(p0, part[0]);
        __syncthreads();
      } else {
        load(step, part[1], ordinary);
        load(step + 1, part[0], ordinary);
        write(p1, part[1]);
        __syncthreads();
        loaded_step(step++, p1, ordinary);
      }
      for (; step + 3 < end; step += 2) {
        loaded_step(step, p0, ordinary);
        loaded_step(step + 1, p1, ordinary);
      }
      loaded_step(step, p0, last);
    }
    multiply(p1, more, part[0]);
    __syncthreads();
  }
  multiply(p0, no_more, part[0]);
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

// 16 bytes of a row from byte k < len on; what lies behind the row's end reads as zero.  At the end the bytes are loaded one
// by one, the last one again in place of those that are not there: sixteen loads in flight, where a branch around each
// would wait for each.
__device__ __forceinline__ u32x4 load_bytes(const int8_t* row, int64_t k, int64_t len) {
  if (k + 16 <= len) return *(const u32x4_align1*)(row + k);
  const int some = (int)(len - k);
  uint32_t byte[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) byte[i] = (uint8_t)row[k + (i < some ? i : some - 1)];
  u32x4 v;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t word = byte[4 * w] | byte[4 * w + 1] << 8 | byte[4 * w + 2] << 16 | byte[4 * w + 3] << 24;
    v[w] = some >= 4 * w + 4 ? word : some <= 4 * w ? 0u : word & ((1u << (8 * (some - 4 * w))) - 1u);
  }
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

// v sa sb + bias.  A sum times a scale from 2^96 on can leave fp32's range where the result does not: the other scale goes first then.
__device__ __forceinline__ bool goes_first(float scale) { return fabsf(scale) < 0x1p96f; }
__device__ __forceinline__ float scaled(int32_t v, float sa, float sb, float bias) {
  return goes_first(sa) ? fmaf((float)v * sa, sb, bias) : fmaf((float)v * sb, sa, bias);
}

// What every tile of the product shares: where it lies, one step's products, and the way out.
template <int DT, int BM, int BN, int WM, int WN>
struct MatmulTile {
  static constexpr int kWaves = WM * WN, kThreads = kWaves * 64, kM = BM / WM / 32, kN = BN / WN / 32;
  using TA = ByteTile<BM, kThreads>;
  using TB = ByteTile<BN, kThreads>;
  const MatmulArgs& p;
  int64_t m0, n0;
  int split, begin, end, left, wave, lane, wm, wn;
  // The weight's rows are the matrix instruction's first operand: a lane then holds four neighbouring channels of a row.
  i32x16 acc[kN][kM];

  __device__ __forceinline__ MatmulTile(const MatmulArgs& args) : p(args) {
    const int tm = (int)((p.m + BM - 1) / BM), tn = (int)((p.n + BN - 1) / BN);
    split = blockIdx.x / (tm * tn);
    const Tile tile = tile_of(blockIdx.x % (tm * tn), tm, tn);
    m0 = (int64_t)tile.row * BM;
    n0 = (int64_t)tile.col * BN;
    wave = wave_id();
    lane = threadIdx.x % 64;
    wm = wave / WN * (BM / WM);
    wn = wave % WN * (BN / WN);
    const int all = (int)((p.k + kStep - 1) / kStep);
    begin = split * p.steps_per_split;
    end = begin + p.steps_per_split < all ? begin + p.steps_per_split : all;
    left = end == all ? (int)(p.k - (int64_t)(all - 1) * kStep) : kStep;  // bytes of the last step that belong to the sum
#pragma unroll
    for (int j = 0; j < kN; ++j)
#pragma unroll
      for (int i = 0; i < kM; ++i) acc[j][i] = i32x16{};
  }
  __device__ __forceinline__ const int8_t* a() const { return p.a + m0 * p.k; }
  __device__ __forceinline__ const int8_t* b() const { return p.b + n0 * p.k; }
  __device__ __forceinline__ int rows_a() const { return (int)(p.m - m0 < BM ? p.m - m0 : BM); }
  __device__ __forceinline__ int rows_b() const { return (int)(p.n - n0 < BN ? p.n - n0 : BN); }

  // what lies behind the sum's end in the last step's tiles is left out
  template <bool LAST>
  __device__ __forceinline__ void multiply(const int8_t* ta, const int8_t* tb) {
    i32x4 fa[2][kM], fb[2][kN];
    auto read = [&](int ks, i32x4(&ra)[kM], i32x4(&rb)[kN]) OPTIMI_INLINE {
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        rb[j] = TB::read(tb, wn + j * 32 + lane % 32, ks * 2 + lane / 32);
        if (LAST && (ks + 1) * 32 > left) rb[j] &= first_bytes(left - ks * 32 - lane / 32 * 16);
      }
#pragma unroll
      for (int i = 0; i < kM; ++i) ra[i] = TA::read(ta, wm + i * 32 + lane % 32, ks * 2 + lane / 32);
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
  }

  // The sums go through LDS 32 rows at a time, so that a lane has eight neighbouring channels to scale and to store.
  using O = OutBlock<32, BN / WN>;
  __device__ __forceinline__ void store(uint32_t* block) {
    using E = Elem<DT>;
    using T = typename E::type;
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
      float sa[O::kTurns];
      bool ordinary = true;
#pragma unroll
      for (int t = 0; t < O::kTurns; ++t) {
        const int64_t m = m0 + wm + i * 32 + O::row(t);
        sa[t] = p.splits == 1 ? p.a_scales[m < p.m ? m : p.m - 1] : 0.0f;
        ordinary &= goes_first(sa[t]);
      }
      // a branch for all of a lane's rows instead of a choice for each number
      auto rows = [&](auto any) OPTIMI_INLINE {
#pragma unroll
        for (int t = 0; t < O::kTurns; ++t) {
          const int64_t m = m0 + wm + i * 32 + O::row(t);
          uint32_t v[8];
          O::get(block, O::row(t), v);
          if (m < p.m && some > 0) {
            if (p.splits > 1) {
              store_some<OPTIMI_F32>((float*)p.partial + ((int64_t)split * p.m + m) * p.n + n, reinterpret_cast<const float(&)[8]>(v), some);
            } else {
              float f[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                if (any.value) f[e] = scaled((int32_t)v[e], sa[t], sb[e], bias[e]);
                else f[e] = fmaf((float)(int32_t)v[e] * sa[t], sb[e], bias[e]);
              }
              store_some<DT>((T*)p.out + m * p.n + n, f, some, whole_lines(p.n, sizeof(T)));
            }
          }
        }
      };
      if (ordinary) rows(std::false_type{});
      else rows(std::true_type{});
      __builtin_amdgcn_wave_barrier();
    }
  }
};

// Rows that start on 16 bytes: two pairs of tiles in LDS, 256 x 256 (eight waves with 128 x 64 sums each, one workgroup a CU) or
// 128 x 128 (four waves with 64 x 64, two workgroups a CU).  A step of 256 x 256 tiles is 64 KiB of copies for 2048 cycles of
// matrix instructions on each SIMD; between two barriers nothing waits but for LDS, whose reads run one slice ahead.
// 8192 x 11008 x 4096: 330 to 345 us from box to box, 2.14 to 2.24 Pop/s; the matrix units are busy for 61 % of the cycles at 1.95 GHz, and the 1376 tiles fill
// 5.4 of 6 rounds.
template <int DT, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64) matmul_kernel(MatmulArgs p) {
  using M = MatmulTile<DT, BM, BN, WM, WN>;
  using TA = typename M::TA;
  using TB = typename M::TB;
  __shared__ __attribute__((aligned(1024))) int8_t a0[BM * kStep], a1[BM * kStep], b0[BN * kStep], b1[BN * kStep];
  M tile(p);
  const uint32_t len = (uint32_t)p.k;
  const Buffer ra = buffer_of(tile.a(), tile.rows_a() * p.k), rb = buffer_of(tile.b(), tile.rows_b() * p.k);
  run_copied(
      tile.begin, tile.end,
      [&](int step, auto which) OPTIMI_INLINE {
        TA::copy(ra, len, step * kStep, which.value ? a1 : a0);
        TB::copy(rb, len, step * kStep, which.value ? b1 : b0);
      },
      [&](auto which, auto last) OPTIMI_INLINE { tile.template multiply<last.value>(which.value ? a1 : a0, which.value ? b1 : b0); });
  // the second pair of tiles is free
  static_assert(M::kWaves / 2 * M::O::kBytes <= BM * kStep && M::kWaves / 2 * M::O::kBytes <= BN * kStep, "half of the waves' blocks fit either tile");
  tile.store((uint32_t*)((tile.wave < M::kWaves / 2 ? a1 : b1) + tile.wave % (M::kWaves / 2) * M::O::kBytes));
}

// Rows that start anywhere, in small tiles.
template <int DT, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64) matmul_loaded_kernel(MatmulArgs p) {
  using M = MatmulTile<DT, BM, BN, WM, WN>;
  using TA = typename M::TA;
  using TB = typename M::TB;
  __shared__ __attribute__((aligned(1024))) int8_t a0[BM * kStep], a1[BM * kStep], b0[BN * kStep], b1[BN * kStep];
  M tile(p);
  struct Part {
    u32x4 a[TA::kPieces], b[TB::kPieces];
  };
  Part part[2];
  const int rows_a = tile.rows_a(), rows_b = tile.rows_b();
  const uint32_t len = (uint32_t)p.k;
  auto load = [&](int step, Part& v, auto last) OPTIMI_INLINE {
    if constexpr (last.value) {
      TA::load_last(tile.a(), rows_a, len, step * kStep, v.a);
      TB::load_last(tile.b(), rows_b, len, step * kStep, v.b);
    } else {
      TA::load(tile.a(), rows_a, len, step * kStep, v.a);
      TB::load(tile.b(), rows_b, len, step * kStep, v.b);
    }
  };
  auto write = [&](auto which, const Part& v) OPTIMI_INLINE {
    TA::store(v.a, which.value ? a1 : a0);
    TB::store(v.b, which.value ? b1 : b0);
  };
  run_loaded(tile.begin, tile.end, part, load, write, [&](auto which, auto more, const Part& v) OPTIMI_INLINE {
    tile.template multiply<false>(which.value ? a1 : a0, which.value ? b1 : b0);
    if (more.value) write(Pair<1 - which.value>{}, v);
  });
  static_assert(M::kWaves / 2 * M::O::kBytes <= BM * kStep && M::kWaves / 2 * M::O::kBytes <= BN * kStep, "half of the waves' blocks fit either tile");
  tile.store((uint32_t*)((tile.wave < M::kWaves / 2 ? a1 : b1) + tile.wave % (M::kWaves / 2) * M::O::kBytes));
}

// Small tiles, for products with less work than the machine has places: a workgroup is alone on its CU or nearly, and
// what counts is that a step does not take a trip to memory.  Four pairs of tiles, three steps on their way: 0.25 us a step,
// 0.38 us with two pairs.  200 x 4096 x 11008: 20 us (two pairs: 41 us), at which its 256 tiles take 18 TB/s from L2; reading the
// operands once from memory would take 10 us.
template <int DT, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64) matmul_deep_kernel(MatmulArgs p) {
  using M = MatmulTile<DT, BM, BN, WM, WN>;
  using TA = typename M::TA;
  using TB = typename M::TB;
  __shared__ __attribute__((aligned(1024))) int8_t a0[BM * kStep], a1[BM * kStep], a2[BM * kStep], a3[BM * kStep];
  __shared__ __attribute__((aligned(1024))) int8_t b0[BN * kStep], b1[BN * kStep], b2[BN * kStep], b3[BN * kStep];
  M tile(p);
  const uint32_t len = (uint32_t)p.k;
  const Buffer ra = buffer_of(tile.a(), tile.rows_a() * p.k), rb = buffer_of(tile.b(), tile.rows_b() * p.k);
  // Steps behind the end are fetched as well, so that the number of copies on their way is always the same; their
  // addresses lie outside of the buffers and nothing is read.
  auto fetch = [&](int step, int8_t* a, int8_t* b) OPTIMI_INLINE {
    const uint32_t k0 = step < tile.end ? (uint32_t)step * kStep : 0x40000000u;
    TA::copy(ra, len, k0, a);
    TB::copy(rb, len, k0, b);
  };
  // This wave's copies but those of the two youngest steps have landed, then everybody's have; the step before is read.
  auto meet_early = [&]() OPTIMI_INLINE {
    constexpr int kYoung = 2 * (TA::kPieces + TB::kPieces);
    static_assert(kYoung == 8, "the count in the instruction below");
    asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  const int begin = tile.begin, end = tile.end;
  if (begin < end) {
    fetch(begin, a0, b0);
    fetch(begin + 1, a1, b1);
    fetch(begin + 2, a2, b2);
    auto one = [&](int at, int8_t* a, int8_t* b, int8_t* next_a, int8_t* next_b, auto last) OPTIMI_INLINE {
      meet_early();
      fetch(at + 3, next_a, next_b);
      __builtin_amdgcn_sched_barrier(0);
      tile.template multiply<last.value>(a, b);
    };
    // rounds of four steps without a branch (the compiler counts the copies in flight by itself too, and a branch makes it
    // wait for more of them than it has to), then the last one to four
    int step = begin;
    for (; step + 4 < end; step += 4) {
      one(step, a0, b0, a3, b3, std::false_type{});
      one(step + 1, a1, b1, a0, b0, std::false_type{});
      one(step + 2, a2, b2, a1, b1, std::false_type{});
      one(step + 3, a3, b3, a2, b2, std::false_type{});
    }
    const int more = end - step;
    if (more > 1) {
      one(step, a0, b0, a3, b3, std::false_type{});
      if (more > 2) {
        one(step + 1, a1, b1, a0, b0, std::false_type{});
        if (more > 3) {
          one(step + 2, a2, b2, a1, b1, std::false_type{});
          one(step + 3, a3, b3, a2, b2, std::true_type{});
        } else {
          one(step + 2, a2, b2, a1, b1, std::true_type{});
        }
      } else {
        one(step + 1, a1, b1, a0, b0, std::true_type{});
      }
    } else {
      one(step, a0, b0, a3, b3, std::true_type{});
    }
  }
  meet();  // all copies have landed and all tiles are read
  static_assert(M::kWaves * M::O::kBytes <= 2 * BM * kStep && M::kWaves / 2 * M::O::kBytes <= BM * kStep, "half of the waves' blocks fit a tile");
  tile.store((uint32_t*)((tile.wave < M::kWaves / 2 ? a0 : a1) + tile.wave % (M::kWaves / 2) * M::O::kBytes));
}

// A few rows against a weight: the weight is read once and nothing else counts.  A wavefront takes kRowsB rows of it, 16
// bytes a lane, multiplies them with up to M rows of the activation, and adds up over its lanes at the end.  KSPLIT
// wavefronts share the same rows of the weight, each a part of the sum, where there are few of them.  1 x 11008 x 4096: 45 MB in
// 7.9 us of kernel, 5.7 TB/s.
constexpr int kRowsB = 4;
struct IntSum {
  static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b) { return a + b; }
};
template <int DT, int M, int KSPLIT>
__global__ void __launch_bounds__(256) matvec_kernel(MatmulArgs p) {
  using E = Elem<DT>;
  using T = typename E::type;
  __shared__ int32_t sums[KSPLIT > 1 ? 4 : 1][kRowsB * M];
  const int wave = wave_id(), lane = threadIdx.x % 64, part = wave % KSPLIT;
  const int64_t n0 = ((int64_t)blockIdx.x * (4 / KSPLIT) + wave / KSPLIT) * kRowsB;
  int32_t acc[kRowsB][M];
#pragma unroll
  for (int r = 0; r < kRowsB; ++r)
#pragma unroll
    for (int m = 0; m < M; ++m) acc[r][m] = 0;
  const int8_t* row[kRowsB];
#pragma unroll
  for (int r = 0; r < kRowsB; ++r) row[r] = p.b + (n0 + r < p.n ? n0 + r : p.n - 1) * p.k;  // rows behind the last: the last again
  auto some = [&](int64_t k, auto whole) OPTIMI_INLINE {
    u32x4 w[kRowsB], x[M];
#pragma unroll
    for (int r = 0; r < kRowsB; ++r) w[r] = whole.value ? *(const u32x4_align1*)(row[r] + k) : load_bytes(row[r], k, p.k);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const int8_t* a = p.a + (m < p.m ? m : p.m - 1) * p.k;
      x[m] = whole.value ? *(const u32x4_align1*)(a + k) : load_bytes(a, k, p.k);
    }
#pragma unroll
    for (int r = 0; r < kRowsB; ++r)
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[r][m] = __builtin_amdgcn_sdot4((int)w[r][i], (int)x[m][i], acc[r][m], false);
  };
  int64_t k = (int64_t)part * 1024 + lane * 16;
#pragma unroll 2
  for (; k + 16 <= p.k; k += KSPLIT * 1024) some(k, std::true_type{});
  if (k < p.k) some(k, std::false_type{});
#pragma unroll
  for (int r = 0; r < kRowsB; ++r)
#pragma unroll
    for (int m = 0; m < M; ++m) acc[r][m] = (int32_t)wave_reduce<IntSum>((uint32_t)acc[r][m]);
  if constexpr (KSPLIT > 1) {
    if (lane == 0) {
#pragma unroll
      for (int r = 0; r < kRowsB; ++r)
#pragma unroll
        for (int m = 0; m < M; ++m) sums[wave][r * M + m] = acc[r][m];
    }
    __syncthreads();
    if (part != 0) return;
  }
  // lane r * M + m stores result (m, n0 + r)
  if (lane >= kRowsB * M) return;
  int32_t sum = 0;
  if constexpr (KSPLIT > 1) {
#pragma unroll
    for (int w = 0; w < KSPLIT; ++w) sum += sums[wave + w][lane];
  } else {
#pragma unroll
    for (int r = 0; r < kRowsB; ++r)
#pragma unroll
      for (int m = 0; m < M; ++m) sum = lane == r * M + m ? acc[r][m] : sum;
  }
  const int64_t m = lane % M, n = n0 + lane / M;
  if (m >= p.m || n >= p.n) return;
  const float bias = p.bias ? E::get(((const T*)p.bias)[n]) : 0.0f;
  ((T*)p.out)[m * p.n + n] = E::put(scaled(sum, p.a_scales[m], p.b_scales[n], bias));
}

// Copies of up to two matrices whose rows of `from` bytes lie `to` bytes apart afterwards, a multiple of 16, with zeros in between: what
// the asynchronous copies need.
struct PadArgs {
  const int8_t* src[2];
  int64_t rows[2];
  uint32_t from, to;
  int8_t* dst;  // the second matrix behind the first
};
__global__ void __launch_bounds__(256) pad_kernel(PadArgs p) {
  const uint32_t pieces = p.to / 16;
  for (int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; row < p.rows[0] + p.rows[1]; row += (int64_t)gridDim.x * 4) {
    const int8_t* src = row < p.rows[0] ? p.src[0] + row * p.from : p.src[1] + (row - p.rows[0]) * p.from;
    for (uint32_t c = threadIdx.x % 64; c < pieces; c += 64) *(u32x4*)(p.dst + row * p.to + c * 16) = load_bytes(src, c * 16, p.from);
  }
}

// Adds the splits' whole-number sums, four neighbours a lane.
template <int DT>
__global__ void __launch_bounds__(256) matmul_finish_kernel(MatmulArgs p) {
  using E = Elem<DT>;
  using T = typename E::type;
  const int64_t all = p.m * p.n;
  for (int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; at < all; at += (int64_t)gridDim.x * 1024) {
    typedef i32x4 i32x4_align4 __attribute__((aligned(4)));
    const int some = (int)(all - at < 4 ? all - at : 4);
    int32_t sum[4] = {0, 0, 0, 0};
    if (some == 4) {
#pragma unroll 4
      for (int s = 0; s < p.splits; ++s) {
        const i32x4 v = *(const i32x4_align4*)(p.partial + s * all + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += v[e];
      }
    } else {
      for (int s = 0; s < p.splits; ++s)
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (e < some) sum[e] += p.partial[s * all + at + e];
    }
    int64_t m = at / p.n, n = at % p.n;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e >= some) break;
      const float bias = p.bias ? E::get(((const T*)p.bias)[n]) : 0.0f;
      ((T*)p.out)[at + e] = E::put(scaled(sum[e], p.a_scales[m], p.b_scales[n], bias));
      if (++n == p.n) {
        n = 0;
        ++m;
      }
    }
  }
}

// ------------------------------------------------------------------------------------
// dw[n][k] = sum_m g[m][n] s[m] q[m][k]
// ------------------------------------------------------------------------------------

struct WeightGradArgs {
  const void* grad;
  int64_t stride;      // of the gradient's rows, in elements
  const int8_t* values;
  const float* scales;
  int64_t rows, outs, cols;
  void* out;
  float* partial;  // [splits][outs][cols] where the sum is split
  int splits;
  int steps_per_split;
  void* bias;           // sums of the gradient over rows, or NULL: by the workgroups of the first columns' tiles, which
  float* bias_partial;  // have all gradients in their hands anyway; [splits][outs] where the sum is split
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

// The upper 8 bits of two fp32 numbers as two bf16 ones; what is left of them stays in x and y.  Three times over, the
// pieces add up to a finite number exactly.
__device__ __forceinline__ uint32_t split_pair(float& x, float& y) {
  const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
  x -= __uint_as_float(a & 0xffff0000u);
  y -= __uint_as_float(b & 0xffff0000u);
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}
// An infinity or a NaN is its own first piece (a NaN stays one without its lower bits) and leaves nothing.
__device__ __forceinline__ uint32_t split_pair_special(float& x, float& y) {
  uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
  x = abs_bits(x) < 0x7f800000u ? x - __uint_as_float(a & 0xffff0000u) : 0.0f;
  y = abs_bits(y) < 0x7f800000u ? y - __uint_as_float(b & 0xffff0000u) : 0.0f;
  a |= (a & 0x7fffffffu) > 0x7f800000u ? 0x400000u : 0u;
  b |= (b & 0x7fffffffu) > 0x7f800000u ? 0x400000u : 0u;
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
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

// Rows 32 ks .. 32 ks + 31 of 16 columns from `offset` on, as the matrix instruction takes them (in an order of rows that is the same
// for both operands).
template <int C>
__device__ __forceinline__ s16x8 read_column(const short* tile, int offset, int ks) {
  typedef OPTIMI_LDS s16x4* Ptr;
  const short* from = tile + offset + ks * 32 * C;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)from);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(from + 16 * C));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Four values as 16-bit numbers; their products with the scale have no rounding under a power of two.
template <int DT>
__device__ __forceinline__ u32x2 widen(uint32_t word, float s) {
  float f[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = (float)(int8_t)(word >> (8 * e)) * s;
  return u32x2{Product<DT>::pair(f[0], f[1]), Product<DT>::pair(f[2], f[3])};
}

// A wave's 16 kN x 16 kC sums, 16 rows at a time through LDS: to the result or, with PARTS where the sum is split, to a part's place.
template <int DT, class O, bool PARTS, int kN, int kC>
__device__ __forceinline__ void store_sums(const WeightGradArgs& p, const f32x4 (&acc)[kN][kC], uint32_t* block, int split, int64_t n0, int64_t c0) {
  using T = typename Elem<DT>::type;
  const int lane = threadIdx.x % 64;
  const int64_t c = c0 + O::col();
  const int64_t some = p.cols - c;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
#pragma unroll
    for (int j = 0; j < kC; ++j) O::put(block, lane % 16, j * 4 + lane / 16, __builtin_bit_cast(u32x4, acc[i][j]));
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int t = 0; t < O::kTurns; ++t) {
      const int64_t n = n0 + i * 16 + O::row(t);
      uint32_t v[8];
      O::get(block, O::row(t), v);
      const float(&f)[8] = reinterpret_cast<const float(&)[8]>(v);
      if (n < p.outs && some > 0) {
        if (PARTS && p.splits > 1) store_some<OPTIMI_F32>(p.partial + ((int64_t)split * p.outs + n) * p.cols + c, f, some);
        else store_some<DT>((T*)p.out + n * p.cols + c, f, some, whole_lines(p.cols, sizeof(T)));
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// 128 x 128 tiles, 64 rows a step, two pairs of tiles in LDS, eight wavefronts with 64 x 32 sums each.  Both operands go through
// registers, from any address: they are loaded two steps ahead, turned into what the matrix instruction takes while
// the step before theirs is multiplied, and written to LDS.  fp32 gradients are multiplied by their row's scale and split into
// three bf16 pieces, so that their products are exact and cost three times as many instructions; the values are
// whole numbers there.  NARROW: rows are shorter than a piece of a load, every load looks at the borders.
// fp32 1000 x 4096 x 1023 with bias: 34.5 us; a step of 64 rows takes 1.7 us, of which the matrix instructions need 0.7 and the
// cutting into pieces about as much.  bf16 2048 x 2048 x 2048: 28 us, 0.65 us a step.
template <int DT, bool NARROW>
__global__ void __launch_bounds__(512) weight_grad_kernel(WeightGradArgs p) {
  using E = Elem<DT>;
  using T = typename E::type;
  using P = Product<DT>;
  constexpr int kTile = 128, kRows = 64, kWaves = 8, kN = 4, kC = 2, kGrad = 2, kPieces = P::kPieces;
  constexpr int kPlane = kRows * kTile;
  using H = HalfTile<kTile>;
  __shared__ __attribute__((aligned(1024))) short g0[kPieces * kPlane], g1[kPieces * kPlane], q0[kPlane], q1[kPlane];
  const int tn = (int)((p.outs + kTile - 1) / kTile), tc = (int)((p.cols + kTile - 1) / kTile);
  const int split = blockIdx.x / (tn * tc);
  const Tile tile = tile_of(blockIdx.x % (tn * tc), tn, tc);
  const int64_t n0 = (int64_t)tile.row * kTile, c0 = (int64_t)tile.col * kTile;
  const int wave = wave_id(), lane = threadIdx.x % 64;
  const int wn = wave / 4 * 64, wc = wave % 4 * 32;
  const int all = (int)((p.rows + kRows - 1) / kRows);
  const int begin = split * p.steps_per_split, end = begin + p.steps_per_split < all ? begin + p.steps_per_split : all;

  f32x4 acc[kN][kC];
#pragma unroll
  for (int i = 0; i < kN; ++i)
#pragma unroll
    for (int j = 0; j < kC; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  // a lane's part of a step: eight gradients of each of two rows, sixteen values of one
  struct Part {
    typename E::Raw g[kGrad];
    float sg[kGrad];
    u32x4 q;
    float sq;
  };
  Part part[2];
  const int outs = (int)(p.outs - n0 < kTile ? p.outs - n0 : kTile), cols = (int)(p.cols - c0 < kTile ? p.cols - c0 : kTile);
  const int g_row = threadIdx.x / 16, g_col = threadIdx.x % 16 * 8, q_row = threadIdx.x / 8, q_col = threadIdx.x % 8 * 16;
  // Columns behind the matrix are read from its first ones and never used; a piece that begins inside may run into the next
  // row, of which there is one in all steps but the last.  The last step's loads look at the borders, and bring zeros from behind them.
  auto load = [&](int step, Part& v, auto last) OPTIMI_INLINE {
    const int64_t m0 = (int64_t)step * kRows;
    const T* grad = (const T*)p.grad + m0 * p.stride + n0;
    const int8_t* values = p.values + m0 * p.cols + c0;
    const float* scales = p.scales + m0;
    if constexpr (!NARROW && !last.value) {
#pragma unroll
      for (int i = 0; i < kGrad; ++i) {
        v.g[i] = E::load(grad + ((uint32_t)(g_row + i * 32) * (uint32_t)p.stride + (g_col < outs ? g_col : 0)));
        if (kPieces > 1) v.sg[i] = scales[g_row + i * 32];
      }
      v.q = *(const u32x4_align1*)(values + ((uint32_t)q_row * (uint32_t)p.cols + (q_col < cols ? q_col : 0)));
      if (kPieces == 1) v.sq = scales[q_row];
    } else {
      const int rows = (int)(p.rows - m0 < kRows ? p.rows - m0 : kRows);
#pragma unroll
      for (int i = 0; i < kGrad; ++i) {
        const bool in = g_row + i * 32 < rows && g_col < outs;
        v.g[i] = E::zero();
        if (in) v.g[i] = load_some<DT>(grad + ((uint32_t)(g_row + i * 32) * (uint32_t)p.stride + g_col), outs - g_col);
        if (kPieces > 1) v.sg[i] = in ? scales[g_row + i * 32] : 0.0f;
      }
      const bool in = q_row < rows && q_col < cols;
      v.q = in ? load_bytes(values + (uint32_t)q_row * (uint32_t)p.cols, q_col, cols) : u32x4{0, 0, 0, 0};
      if (kPieces == 1) v.sq = in ? scales[q_row] : 0.0f;
    }
  };
  // Turning a part into 16-bit tiles, in as many pieces of work as a step has groups of products, between which they go.  Of
  // an fp32 row's eight numbers two at a time give their next bf16 piece, and after the fourth pair that piece is written.
  constexpr int kGroups = 2 * kPieces * kN;  // groups of kC products in a step
  struct Turn {
    float f[8];
    u32x4 w, q[2];
    uint32_t most;
  };
  auto grad_place = [&](int i, short* g) OPTIMI_INLINE { return g + H::at(g_row + i * 32, g_col / 16) + g_col % 16; };
  auto turn_values = [&](int word, const Part& v, Turn& t, short* q) OPTIMI_INLINE {
    const u32x2 two = widen<DT>(v.q[word], kPieces > 1 ? 1.0f : v.sq);
    t.q[word / 2][word % 2 * 2] = two[0];
    t.q[word / 2][word % 2 * 2 + 1] = two[1];
    if (word % 2) *(u32x4*)(q + H::at(q_row, q_col / 16) + word / 2 * 8) = t.q[word / 2];
  };
  auto turn = [&](int at, const Part& v, Turn& t, short* g, short* q) OPTIMI_INLINE {
    if constexpr (kPieces == 1) {
      if (at < kGrad) *(u32x4*)grad_place(at, g) = v.g[at].a;
      if (at >= kGroups - 4) turn_values(at - (kGroups - 4), v, t, q);
    } else {
      const int i = at / 12, z = at % 12 / 4, e = at % 4;  // the row, the piece, the pair
      if (at % 12 == 0) {
        E::unpack(v.g[i], t.f);
        if (i == 0) t.most = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          t.f[k] *= v.sg[i];
          t.most = MaxOp::join(t.most, abs_bits(t.f[k]));
        }
      }
      t.w[e] = split_pair(t.f[2 * e], t.f[2 * e + 1]);
      if (e == 3) *(u32x4*)(grad_place(i, g) + z * kPlane) = t.w;
      if (at % 6 == 5) turn_values(at / 6, v, t, q);
    }
  };
  // The rows that hold an infinity or a NaN again: such a number leaves nothing to its further pieces.
  auto turn_special = [&](const Part& v, const Turn& t, short* g) OPTIMI_INLINE {
    if constexpr (kPieces > 1) {
      if (t.most < 0x7f800000u) return;
#pragma unroll
      for (int i = 0; i < kGrad; ++i) {
        float f[8];
        E::unpack(v.g[i], f);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] *= v.sg[i];
#pragma unroll
        for (int z = 0; z < kPieces; ++z) {
          u32x4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = split_pair_special(f[2 * e], f[2 * e + 1]);
          *(u32x4*)(grad_place(i, g) + z * kPlane) = w;
        }
      }
    }
  };
  const bool with_bias = p.bias && tile.col == 0;
  float bias[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  auto add_bias = [&](const Part& v) OPTIMI_INLINE {
    if (!with_bias) return;
#pragma unroll
    for (int i = 0; i < kGrad; ++i) {
      float f[8];
      E::unpack(v.g[i], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) bias[e] += f[e];
    }
  };
  auto multiply = [&](auto which, auto more, const Part& v) OPTIMI_INLINE {
    const short *g = which.value ? g1 : g0, *q = which.value ? q1 : q0;
    short *next_g = which.value ? g0 : g1, *next_q = which.value ? q0 : q1;
    s16x8 fq[2][kC], fg[3];
    Turn t;
    auto read_g = [&](int at) OPTIMI_INLINE {  // the smallest pieces first
      const int ks = at / (kGroups / 2), z = kPieces - 1 - at % (kGroups / 2) / kN, i = at % kN;
      return read_column<kTile>(g + z * kPlane, H::at(lane / 4, wn / 16 + i) + lane % 4 * 4, ks);
    };
    auto read_q = [&](int ks) OPTIMI_INLINE {
#pragma unroll
      for (int j = 0; j < kC; ++j) fq[ks][j] = read_column<kTile>(q, H::at(lane / 4, wc / 16 + j) + lane % 4 * 4, ks);
    };
    read_q(0);
    fg[0] = read_g(0);
    fg[1] = read_g(1);
#pragma unroll
    for (int at = 0; at < kGroups; ++at) {
      if (at + 2 < kGroups) fg[(at + 2) % 3] = read_g(at + 2);
      if (at == kGroups / 2 - 2) read_q(1);
#pragma unroll
      for (int j = 0; j < kC; ++j) acc[at % kN][j] = P::mfma(fq[at / (kGroups / 2)][j], fg[at % 3], acc[at % kN][j]);
      if (more.value) turn(at, v, t, next_g, next_q);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (more.value) {
      turn_special(v, t, next_g);
      add_bias(v);
    }
  };
  run_loaded(begin, end, part, load,
             [&](auto which, const Part& v) OPTIMI_INLINE {
               Turn t;
#pragma unroll
               for (int at = 0; at < kGroups; ++at) turn(at, v, t, which.value ? g1 : g0, which.value ? q1 : q0);
               turn_special(v, t, which.value ? g1 : g0);
               add_bias(v);
             },
             multiply);
  if (with_bias) {  // 32 lanes have sums of the same columns
    float* sums = (float*)g0;
    static_assert(32 * kTile * 4 <= kPlane * 2, "the sums fit a tile");
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[g_row * kTile + g_col + e] = bias[e];
    __syncthreads();
    const int64_t n = n0 + threadIdx.x;
    if (threadIdx.x < kTile && n < p.outs) {
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 32; ++r) sum += sums[r * kTile + threadIdx.x];
      if (p.splits > 1) p.bias_partial[split * p.outs + n] = sum;
      else ((T*)p.bias)[n] = E::put(sum);
    }
  }

  using O = OutBlock<16, 32>;
  static_assert(kWaves / 2 * O::kBytes <= kPlane * 2, "half of the waves' blocks fit a tile");
  store_sums<DT, O, true, kN, kC>(p, acc, (uint32_t*)((char*)(wave < 4 ? g1 : q1) + wave % 4 * O::kBytes), split, n0 + wn, c0 + wc);
}

// The same for large 16-bit products, where all that counts is that the matrix instructions never wait: 256 x 256 tiles, 64
// rows a step, two pairs of tiles in LDS, eight wavefronts with 128 x 64 sums each.  Gradients go to LDS past the registers;
// the values have to become 16-bit numbers on the way, and are loaded two steps ahead, so that the conversion of the next
// step's values can be spread over this step's products without waiting for memory.  outs is a multiple of 8, grad aligned to
// 16 bytes, a row has 16 values at least, and there are more than 128 tiles: their sums are never split.
//
// 8192 x 11008 x 4096 bf16: 672 us among passes over changing inputs, 1.10 PFLOP/s; on one set of inputs in a row 648 us, where a library's
// bf16 product of the same gradients and of the values widened beforehand takes 760; a step takes 3900 busy cycles by the counters, of which the matrix units are busy for 2048, LDS for 1300 (a
// fifth of them bank conflicts) and vector instructions for 1000, two thirds of them the conversion: ten for four values (with eleven, and
// the last step's borders worked out in every step, 735 us); 688 tiles fill 2.7 of 3 rounds.  A raised wave priority around the products changes nothing.
template <int DT>
__global__ void __launch_bounds__(512) weight_grad_wide_kernel(WeightGradArgs p) {
  using T = typename Elem<DT>::type;
  using P = Product<DT>;
  constexpr int kTile = 256, kRows = 64, kN = 8, kC = 4, kPieces = 2;
  using H = HalfTile<kTile>;
  __shared__ __attribute__((aligned(1024))) short g0[kRows * kTile], g1[kRows * kTile], q0[kRows * kTile], q1[kRows * kTile];
  const int tn = (int)((p.outs + kTile - 1) / kTile), tc = (int)((p.cols + kTile - 1) / kTile);
  const Tile tile = tile_of(blockIdx.x, tn, tc);
  const int64_t n0 = (int64_t)tile.row * kTile, c0 = (int64_t)tile.col * kTile;
  const int wave = wave_id(), lane = threadIdx.x % 64;
  const int wn = wave / 4 * 128, wc = wave % 4 * 64;
  const int all = (int)((p.rows + kRows - 1) / kRows);

  f32x4 acc[kN][kC];
#pragma unroll
  for (int i = 0; i < kN; ++i)
#pragma unroll
    for (int j = 0; j < kC; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  // Gradients: a wave's copy fills two rows of LDS; the sources follow the swizzle.  Columns behind the matrix come from the
  // next row (or not at all, behind the last) and end in sums that are not stored.  What the last step has less than the
  // others is worked out once and chosen inside the loop: 683 us instead of 707 at 8192 x 11008 x 4096.
  const int last_rows = (int)(p.rows - (int64_t)(all - 1) * kRows);
  auto rows_of = [&](int step) OPTIMI_INLINE { return step + 1 == all ? last_rows : kRows; };
  const uint32_t width = (uint32_t)(p.stride - n0 < kTile ? p.stride - n0 : kTile);
  auto copy = [&](int step, short* g) OPTIMI_INLINE {
    const T* base = (const T*)p.grad + (int64_t)step * kRows * p.stride + n0;
    const uint32_t bytes = ((uint32_t)(rows_of(step) - 1) * (uint32_t)p.stride + width) * 2;  // below 2^31: see kMostWidth
    const Buffer from = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, (int)bytes, 0x00020000);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int place = i * 512 + threadIdx.x;
      const int row = place / 32, in = place % 32;
      const int n = H::at(row, in / 2) - row * kTile + in % 2 * 8;
      copy16_to_lds(from, ((uint32_t)row * (uint32_t)p.stride + n) * 2, g + (i * 512 + wave * 64) * 8);
    }
  };
  // Values: a lane has 16 neighbours of two rows.  Rows behind the last are the last one again, under a scale of 0;
  // columns behind the matrix are never used.  A piece that would run over the end of all values - in the last step only, the
  // others have a row of 16 values at least behind them - is loaded from a little before, and shifted into its place
  // when it is converted.
  const int64_t total = p.rows * p.cols;
  const int at_row = threadIdx.x / 16, at_col = threadIdx.x % 16;
  const uint32_t col = (uint32_t)c0 + (c0 + at_col * 16 < p.cols ? at_col * 16 : 0);
  u32x4 vq[2][kPieces];
  float sq[2][kPieces];
  const int64_t last_first = (int64_t)(all - 1) * kRows * p.cols, last_start = last_first < total - 16 ? last_first : total - 16;
  const uint32_t last_limit = (uint32_t)(total - 16 - last_start);
  auto place_of = [&](int step, int i, int64_t& start, uint32_t& limit) OPTIMI_INLINE {
    const int64_t first = (int64_t)step * kRows * p.cols;
    const bool is_last = step + 1 == all;
    start = is_last ? last_start : first;
    limit = is_last ? last_limit : 0x7fffffffu;
    const int rows = rows_of(step), row = at_row + i * 32;
    return (uint32_t)(row < rows ? row : rows - 1) * (uint32_t)p.cols + col + (uint32_t)(first - start);
  };
  auto load = [&](int step, u32x4 (&v)[kPieces], float (&s)[kPieces]) OPTIMI_INLINE {
    const int64_t m0 = (int64_t)step * kRows;
    const int rows = rows_of(step);
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
  auto shift = [&](int step, u32x4 (&v)[kPieces], float (&s)[kPieces]) OPTIMI_INLINE {  // the very last step only
    const int rows = rows_of(step);
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
  auto write_half = [&](int half, const u32x4 (&v)[kPieces], const float (&s)[kPieces], short* q) OPTIMI_INLINE {  // eight values of piece half / 2
    const int i = half / 2;
    const u32x2 a = widen<DT>(v[i][half % 2 * 2], s[i]), b = widen<DT>(v[i][half % 2 * 2 + 1], s[i]);
    *(u32x4*)(q + H::at(at_row + i * 32, at_col) + half % 2 * 8) = u32x4{a[0], a[1], b[0], b[1]};
  };

  // Where a lane's part of 16 columns lies: chunks differ in five address bits only, so chunk i of the wave's is one
  // exclusive or away from its first.  The addresses are formed anew for every step: kept over the loop, they would take more
  // registers than there are.
  typedef OPTIMI_LDS s16x4* Ptr;
  auto column = [&](const short* t, int first, int i, int ks) OPTIMI_INLINE {
    const char* from = (const char*)t + (first ^ (i * 32)) + ks * 32 * kTile * 2;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)from);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(from + 16 * kTile * 2));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto anew = [](int v) OPTIMI_INLINE {
    asm volatile("" : "+v"(v));
    return v & 0x7fff;
  };
  const int first_g = (H::at(lane / 4, wn / 16) + lane % 4 * 4) * 2, first_q = (H::at(lane / 4, wc / 16) + lane % 4 * 4) * 2;
  // One step's products in sixteen groups; a group's operands are read two groups earlier, and four of the groups are followed
  // by a quarter of the next step's conversion.
  auto multiply = [&](const short* g, const short* q, auto last, const u32x4 (&v)[kPieces], const float (&s)[kPieces], short* next) OPTIMI_INLINE {
    const int at_g = anew(first_g), at_q = anew(first_q);
    s16x8 fq[2][kC], fg[3];
    auto keep = [&](s16x8 f, int ks) OPTIMI_INLINE {  // copied gradients of rows behind the last are whatever was in LDS, infinities maybe
      if (!last.value) return f;
      s16x8 mask;
#pragma unroll
      for (int e = 0; e < 8; ++e) mask[e] = ks * 32 + e / 4 * 16 + lane / 16 * 4 + e % 4 < last_rows ? -1 : 0;
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
  auto step_on = [&](int step, auto which) OPTIMI_INLINE {
    constexpr int W = decltype(which)::value;
    copy(step + 1, W ? g0 : g1);
    if (step + 2 < all) load(step + 2, vq[W], sq[W]);
    if (step + 2 == all) shift(step + 1, vq[1 - W], sq[1 - W]);
    __builtin_amdgcn_sched_barrier(0);  // the loads start before the products do; left alone, they are moved behind them
    multiply(W ? g1 : g0, W ? q1 : q0, std::false_type{}, vq[1 - W], sq[1 - W], W ? q0 : q1);
    meet();
  };
  auto start = [&](int step, auto which) OPTIMI_INLINE {
    constexpr int W = decltype(which)::value;
    copy(step, W ? g1 : g0);
    load(step, vq[W], sq[W]);
    if (step + 1 < all) load(step + 1, vq[1 - W], sq[1 - W]);
    if (step + 1 == all) shift(step, vq[W], sq[W]);
#pragma unroll
    for (int half = 0; half < 2 * kPieces; ++half) write_half(half, vq[W], sq[W], W ? q1 : q0);
    meet();
  };

  // the last step works on the first pair of tiles
  int step = 0;
  if (all % 2) {
    start(step, Pair<0>{});
  } else {
    start(step, Pair<1>{});
    step_on(step++, Pair<1>{});
  }
  for (; step + 1 < all; step += 2) {
    step_on(step, Pair<0>{});
    step_on(step + 1, Pair<1>{});
  }
  multiply(g0, q0, std::true_type{}, vq[0], sq[0], q1);

  using O = OutBlock<16, 64>;
  store_sums<DT, O, false, kN, kC>(p, acc, (uint32_t*)((char*)(wave < 4 ? g1 : q1) + wave % 4 * O::kBytes), 0, n0 + wn, c0 + wc);
}

// Adds the splits' sums, four neighbours a lane, always in the same order.
template <int DT>
__global__ void __launch_bounds__(256) weight_grad_finish_kernel(WeightGradArgs p) {
  using E = Elem<DT>;
  typedef f32x4 f32x4_align4 __attribute__((aligned(4)));
  const int64_t n = p.outs * p.cols;
  for (int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; at < n; at += (int64_t)gridDim.x * 1024) {
    const int some = (int)(n - at < 4 ? n - at : 4);
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (some == 4) {
#pragma unroll 8
      for (int s = 0; s < p.splits; ++s) {
        const f32x4 v = *(const f32x4_align4*)(p.partial + s * n + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += v[e];
      }
    } else {
      for (int s = 0; s < p.splits; ++s)
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (e < some) sum[e] += p.partial[s * n + at + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < some) ((typename E::type*)p.out)[at + e] = E::put(sum[e]);
  }
}

constexpr int64_t kMostWidth = 1 << 24;  // of a weight gradient: offsets inside a tile stay in 31 bits
constexpr int64_t kMostSum = 131071;  // (-128)^2 times this stays below 2^31
// A launch holds fewer than 2^32 lanes.
inline bool launch_holds(int64_t workgroups, int lanes) { return workgroups < ((int64_t)1 << 32) / lanes; }

// How a product is cut: the tile's size and the number of parts that the sum is split into.
struct Cut {
  int tile;
  int64_t tiles;
  int splits, steps_per_split;
  void split(int64_t steps, int64_t parts) {
    splits = parts > 1 ? (int)parts : 1;
    steps_per_split = (int)((steps + splits - 1) / splits);
    if (splits > 1) splits = (int)((steps + steps_per_split - 1) / steps_per_split);
  }
};
constexpr int kCus = 256;
inline int64_t tiles_of(int64_t rows, int64_t cols, int tile) { return ((rows + tile - 1) / tile) * ((cols + tile - 1) / tile); }

// Which tile: the one whose steps, for all of its tiles, take the least time.  Measured in microseconds per step of 128 bytes on
// the whole machine, int8 operands that come from the caches: 256 x 256 tiles 1.55 where they leave half of the 256 CUs empty,
// 2.05 per round of 256; 128 x 128 tiles 0.68, 0.82 up to one per CU, 1.2 per round of two per CU; 64 x 64 tiles 0.25 up to
// one per CU, then 0.22 for each further one.  (2048 x 4096 x 4096: 52 us in tiles of 256, 41 in tiles of 128, 60 in
// tiles of 64; 4096 x 4096 x 4096: 66, 77, 112; 512 x 4096 x 4096: 47, 24, 18.)  Few tiles with a long sum are split into parts
// for the idle CUs where that saves more than the joining launch costs, 3.5 us and the partial sums' way to memory and back:
// 100 x 100 x 16384 takes 23 us whole and 9.2 us in 16 parts, 64 x 4096 x 4096 9.1 us whole and 10.9 us in four.
Cut matmul_cut(int64_t m, int64_t n, int64_t k) {
  const int64_t steps = (k + kStep - 1) / kStep;
  const int64_t t256 = tiles_of(m, n, 256), t128 = tiles_of(m, n, 128), t64 = tiles_of(m, n, 64);
  const double c256 = t256 <= kCus / 2 ? 1.55 : 2.05 * (double)((t256 + kCus - 1) / kCus);
  const double c128 = t128 <= kCus / 2 ? 0.68 : t128 <= kCus ? 0.82 : 1.2 * (double)((t128 + 2 * kCus - 1) / (2 * kCus));
  const double c64 = t64 <= kCus ? 0.25 : 0.05 + 0.22 * (double)t64 / kCus;
  Cut c;
  c.tile = c256 <= c128 && c256 <= c64 ? 256 : c128 <= c64 ? 128 : 64;
  c.tiles = c.tile == 256 ? t256 : c.tile == 128 ? t128 : t64;
  int64_t parts = 1;
  if (c.tile == 64) {
    double least = 0.25 * (double)steps;
    for (int64_t s = 2; s <= 16 && s * c.tiles <= kCus && 4 * s <= steps; ++s) {
      const double cost = 0.25 * (double)((steps + s - 1) / s) + 3.5 + (double)s * (double)m * (double)n * 8 / 3e6;
      if (cost < least) {
        least = cost;
        parts = s;
      }
    }
  }
  c.split(steps, parts);
  return c;
}
// The same for weight gradients, in microseconds per step of 64 rows: 2.2 per round of 256 wide tiles; 0.8 for up to 256 tiles
// of 128 x 128, 1.45 per round of two per CU.  (1024 x 4096 x 4096: 43 us in wide tiles, 61 in the others; 2048 x 2048 x 2048:
// 66, 28.)  Four steps at least to a part: 4096 x 512 x 512 takes 44 us whole, 17 us in eight parts.
Cut weight_grad_cut(int64_t rows, int64_t outs, int64_t cols, int dtype) {
  const bool narrow = outs < 8 || cols < 16;
  const int64_t steps = (rows + 63) / 64;
  Cut c;
  const int64_t t256 = tiles_of(outs, cols, 256), t128 = tiles_of(outs, cols, 128);
  const double c256 = 2.2 * (double)((t256 + kCus - 1) / kCus);
  const double c128 = t128 <= kCus ? 0.8 : 1.45 * (double)((t128 + 2 * kCus - 1) / (2 * kCus));
  const bool wide = dtype != OPTIMI_F32 && !narrow && rows * cols >= 16;
  c.tile = wide && c256 <= c128 ? 256 : 128;  // 129 wide tiles at least: where that holds, t128 is above 512
  c.tiles = tiles_of(outs, cols, c.tile);
  int64_t parts = 1;
  if (c.tile == 128 && c.tiles < kCus) parts = kCus / c.tiles < steps / 4 ? kCus / c.tiles : steps / 4;
  c.split(steps, parts < 16 ? parts : 16);
  return c;
}

// Products of at most this many rows are read off the weight without tiles.  (1 x 11008 x 4096: 9.2 us, in tiles 14; 4 x 11008
// x 4096: 9.3 us; 8 x 11008 x 4096: 15.5 us, in tiles 10.2.)
constexpr int64_t kMostVec = 4;
// Bytes that padded copies of the operands take, for rows that do not start on 16 bytes in tiles that are copied asynchronously.
inline int64_t padded(int64_t bytes) { return (bytes + 15) / 16 * 16; }

// What a product of these sizes does: computed alike by the call and by its workspace function.
//
// Odd widths: large tiles are copied asynchronously and take padded copies of both operands.  Small ones can be loaded through registers,
// at 0.44 us a step instead of 0.17 to 0.20 (517 x 1001 and 1000 x 1000, k from 1024 to 8192); the copies cost a launch and 0.5 us per million
// bytes (42 x 216 x 3675: 16.6 us through registers, 13.3 us padded; 20 x 8000 x 8001: 32 us, 38 us).
inline int64_t vec_blocks(int64_t n, bool share) { return share ? (n + 3) / 4 : (n + 15) / 16; }
struct MatmulPlan {
  bool vec;         // read off the weight
  bool pad;         // padded copies of both operands come first
  Cut cut;
  int64_t pad_bytes, partial_bytes;
};
MatmulPlan matmul_plan(int64_t m, int64_t n, int64_t k) {
  MatmulPlan plan{};
  plan.vec = m <= kMostVec && launch_holds(vec_blocks(n, false), 256);
  if (plan.vec) return plan;
  plan.cut = matmul_cut(m, n, k);
  plan.pad = k % 16 != 0 && (plan.cut.tile > 64 || 0.25 * (double)((k + kStep - 1) / kStep) > 2.0 + 0.5e-6 * (double)((m + n) * k));
  plan.pad_bytes = plan.pad ? (m + n) * padded(k) : 0;
  plan.partial_bytes = plan.cut.splits > 1 ? plan.cut.splits * m * n * 4 : 0;
  return plan;
}

inline int matmul_lanes(int tile) { return tile == 256 ? 512 : 256; }

// The sizes that the call and its workspace function refuse.
int matmul_sizes(int64_t m, int64_t n, int64_t k) {
  if (int rc = check_shape(m, n)) return rc;
  if (k < 0 || k > kMostSum) return OPTIMI_ERR_SIZE;
  if (m == 0 || n == 0) return 0;
  const MatmulPlan plan = matmul_plan(m, n, k);
  return plan.vec || launch_holds(plan.cut.tiles * plan.cut.splits, matmul_lanes(plan.cut.tile)) ? 0 : (int)OPTIMI_ERR_SIZE;
}

struct WeightGradPlan {
  bool pad;       // a padded copy of the gradient comes first
  bool bias_own;  // the bias gradient takes launches of its own
  Cut cut;
  int64_t pad_bytes, partial_bytes, bias_bytes;
};
WeightGradPlan weight_grad_plan(int64_t rows, int64_t outs, int64_t cols, int dtype, bool with_bias) {
  WeightGradPlan plan{};
  if (cols > 0) {
    plan.cut = weight_grad_cut(rows, outs, cols, dtype);
    plan.pad = plan.cut.tile == 256 && outs % 8 != 0;
    plan.pad_bytes = plan.pad ? rows * padded(outs * 2) : 0;
    plan.partial_bytes = plan.cut.splits > 1 ? padded(plan.cut.splits * outs * cols * 4) : 0;
  }
  plan.bias_own = with_bias && (cols == 0 || plan.cut.tile == 256);
  if (plan.bias_own) plan.bias_bytes = padded(column_sum_workspace(rows, outs));
  else if (with_bias && plan.cut.splits > 1) plan.bias_bytes = padded(plan.cut.splits * outs * 4);
  return plan;
}

constexpr int kWeightGradLanes = 512;
int weight_grad_sizes(int64_t rows, int64_t outs, int64_t cols, int dtype, bool with_bias) {
  if (int rc = check_shape(rows, outs)) return rc;
  if (int rc = check_shape(rows, cols)) return rc;
  if (outs > kMostWidth || cols > kMostWidth) return OPTIMI_ERR_SIZE;
  if (outs == 0 || cols == 0) return 0;
  const WeightGradPlan plan = weight_grad_plan(rows, outs, cols, dtype, with_bias);
  return launch_holds(plan.cut.tiles * plan.cut.splits, kWeightGradLanes) ? 0 : (int)OPTIMI_ERR_SIZE;
}

template <int DT>
int launch_vec(const MatmulArgs& args, hipStream_t stream) {
  const bool share = (args.n + 15) / 16 < 2 * kCus && args.k > 1024;
  const dim3 grid((unsigned)vec_blocks(args.n, share)), block(256);
  auto go = [&](auto m) {
    constexpr int M = decltype(m)::value;
    if (share) matvec_kernel<DT, M, 4><<<grid, block, 0, stream>>>(args);
    else matvec_kernel<DT, M, 1><<<grid, block, 0, stream>>>(args);
  };
  if (args.m == 1) go(Pair<1>{});
  else if (args.m == 2) go(Pair<2>{});
  else go(Pair<4>{});
  OPTIMI_INT8_TRY(hipGetLastError());
  return 0;
}

int pad_rows(const void* a, int64_t rows_a, const void* b, int64_t rows_b, int64_t from, void* dst, hipStream_t stream) {
  const int64_t blocks = (rows_a + rows_b + 3) / 4;
  const PadArgs args{{(const int8_t*)a, (const int8_t*)b}, {rows_a, rows_b}, (uint32_t)from, (uint32_t)padded(from), (int8_t*)dst};
  pad_kernel<<<dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, stream>>>(args);
  OPTIMI_INT8_TRY(hipGetLastError());
  return 0;
}

}  // namespace

extern "C" {

int64_t optimi_hip_int8_matmul_workspace(int64_t m, int64_t n, int64_t k) {
  if (int rc = matmul_sizes(m, n, k)) return rc;
  if (m == 0 || n == 0) return 0;
  const MatmulPlan plan = matmul_plan(m, n, k);
  return plan.pad_bytes + plan.partial_bytes;
}

int optimi_hip_int8_matmul(const int8_t* a, const float* a_scales, const int8_t* b, const float* b_scales, const void* bias, int64_t m, int64_t n,
                           int64_t k, int dtype, void* out, void* workspace, optimi_stream_t stream_) {
  if (!valid_dtype(dtype)) return OPTIMI_ERR_DTYPE;
  if (int rc = matmul_sizes(m, n, k)) return rc;
  if (m == 0 || n == 0) return 0;
  if (!a_scales || !b_scales || !out || (k && (!a || !b))) return OPTIMI_ERR_NULL;
  const int64_t size = elem_bytes(dtype);
  if (!aligned_to(a_scales, 4) || !aligned_to(b_scales, 4) || !aligned_to(bias, size) || !aligned_to(out, size) || !aligned_to(workspace, 16)) return OPTIMI_ERR_ALIGN;
  const MatmulPlan plan = matmul_plan(m, n, k);
  if (plan.pad_bytes + plan.partial_bytes > 0 && !workspace) return OPTIMI_ERR_NULL;
  hipStream_t stream = (hipStream_t)stream_;
  MatmulArgs args{a, a_scales, b, b_scales, bias, m, n, k, out, nullptr, 1, 0};
  if (plan.vec) return by_dtype(dtype, [&](auto dt) { return launch_vec<decltype(dt)::value>(args, stream); });

  Cut c = plan.cut;
  if (plan.pad) {
    int8_t* pa = (int8_t*)workspace;
    int8_t* pb = pa + m * padded(k);
    if (int rc = pad_rows(a, m, b, n, k, pa, stream)) return rc;
    args.a = pa;
    args.b = pb;
    args.k = padded(k);
  }
  const bool aligned = args.k % 16 == 0 && aligned_to(args.a, 16) && aligned_to(args.b, 16);
  if (!aligned && c.tile > 64) {  // operands that start off the grid: tiles that go through registers are small ones
    c.tile = 64;
    c.tiles = tiles_of(m, n, 64);
    if (!launch_holds(c.tiles * c.splits, matmul_lanes(64))) return OPTIMI_ERR_ALIGN;
  }
  args.partial = (int32_t*)((int8_t*)workspace + plan.pad_bytes);
  args.splits = c.splits;
  args.steps_per_split = c.steps_per_split;
  return by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const dim3 grid((unsigned)(c.tiles * c.splits));
    if (c.tile == 256) {
      matmul_kernel<DT, 256, 256, 2, 4><<<grid, dim3(512), 0, stream>>>(args);
    } else if (c.tile == 128) {
      matmul_kernel<DT, 128, 128, 2, 2><<<grid, dim3(256), 0, stream>>>(args);
    } else {
      if (aligned) matmul_deep_kernel<DT, 64, 64, 2, 2><<<grid, dim3(256), 0, stream>>>(args);
      else matmul_loaded_kernel<DT, 64, 64, 2, 2><<<grid, dim3(256), 0, stream>>>(args);
    }
    OPTIMI_INT8_TRY(hipGetLastError());
    if (c.splits > 1) {
      const int64_t blocks = (m * n + 1023) / 1024;
      matmul_finish_kernel<DT><<<dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, stream>>>(args);
      OPTIMI_INT8_TRY(hipGetLastError());
    }
    return 0;
  });
}

int64_t optimi_hip_int8_weight_grad_workspace(int64_t rows, int64_t outs, int64_t cols, int dtype, int with_bias) {
  if (!valid_dtype(dtype)) return OPTIMI_ERR_DTYPE;
  if (int rc = weight_grad_sizes(rows, outs, cols, dtype, with_bias != 0)) return rc;
  if (outs == 0) return 0;
  const WeightGradPlan plan = weight_grad_plan(rows, outs, cols, dtype, with_bias != 0);
  return plan.pad_bytes + plan.partial_bytes + plan.bias_bytes;
}

int optimi_hip_int8_weight_grad(const void* grad, const int8_t* values, const float* scales, int64_t rows, int64_t outs, int64_t cols, int dtype,
                                void* weight_grad, void* bias_grad, void* workspace, optimi_stream_t stream_) {
  if (!valid_dtype(dtype)) return OPTIMI_ERR_DTYPE;
  if (int rc = weight_grad_sizes(rows, outs, cols, dtype, bias_grad != nullptr)) return rc;
  if (outs == 0) return 0;
  if ((cols && !weight_grad) || (rows && (!grad || (cols && (!scales || !values))))) return OPTIMI_ERR_NULL;
  const int64_t size = elem_bytes(dtype);
  if (!aligned_to(grad, size) || !aligned_to(scales, 4) || !aligned_to(weight_grad, size) || !aligned_to(bias_grad, size) || !aligned_to(workspace, 16))
    return OPTIMI_ERR_ALIGN;
  const WeightGradPlan plan = weight_grad_plan(rows, outs, cols, dtype, bias_grad != nullptr);
  if (plan.pad_bytes + plan.partial_bytes + plan.bias_bytes > 0 && !workspace) return OPTIMI_ERR_NULL;
  hipStream_t stream = (hipStream_t)stream_;
  int8_t* work = (int8_t*)workspace;
  float* bias_work = (float*)(work + plan.pad_bytes + plan.partial_bytes);
  if (plan.bias_own) {
    if (int rc = column_sum(grad, rows, outs, dtype, bias_grad, bias_work, stream)) return rc;
  }
  if (cols == 0) return 0;
  Cut c = plan.cut;
  WeightGradArgs args{grad, outs, values, scales, rows, outs, cols, weight_grad, (float*)(work + plan.pad_bytes), c.splits, c.steps_per_split,
                      plan.bias_own ? nullptr : bias_grad, bias_work};
  if (plan.pad) {
    if (int rc = pad_rows(grad, rows, nullptr, 0, outs * 2, work, stream)) return rc;
    args.grad = work;
    args.stride = padded(outs * 2) / 2;
  }
  const bool direct = args.stride % 8 == 0 && aligned_to(args.grad, 16);
  if (c.tile == 256 && !direct) {
    c.tile = 128;
    c.tiles = tiles_of(outs, cols, 128);
    if (!launch_holds(c.tiles * c.splits, kWeightGradLanes)) return OPTIMI_ERR_ALIGN;
  }
  return by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const dim3 grid((unsigned)(c.tiles * c.splits));
    if (c.tile == 256) {
      if constexpr (DT != OPTIMI_F32) weight_grad_wide_kernel<DT><<<grid, dim3(512), 0, stream>>>(args);
    } else if (outs < 8 || cols < 16) {  // too narrow for whole pieces
      weight_grad_kernel<DT, true><<<grid, dim3(512), 0, stream>>>(args);
    } else {
      weight_grad_kernel<DT, false><<<grid, dim3(512), 0, stream>>>(args);
    }
    OPTIMI_INT8_TRY(hipGetLastError());
    if (c.splits > 1) {
      const int64_t blocks = (outs * cols + 1023) / 1024;
      weight_grad_finish_kernel<DT><<<dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, stream>>>(args);
      OPTIMI_INT8_TRY(hipGetLastError());
      if (args.bias) return finish_columns(bias_work, c.splits, outs, dtype, bias_grad, stream);
    }
    return 0;
  });
}

}  // extern "C"
