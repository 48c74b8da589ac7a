// Row kernels of the int8 activations for MI355X (gfx950): quantize, dequantize, the residual add with RMS norm
// and int8 output, and its backward pass.
//
// All of them stream: every input is read once, every output written once, and HBM bandwidth is the bound.  What
// stands in the way is that a row's scale (and the norm's 1/rms) is known only after the whole row was seen.  A row
// therefore stays in the registers of the team of lanes that works on it - one wavefront for rows of up to 1024 elements, a
// workgroup of four for up to 8192, of eight for up to 16384 - between the reduction and the use of its result; only rows beyond
// 16384 elements are read again (the second read is served by L2).  Sums, the norm's statistics and the quantized values are
// formed in fp32 whatever the type of the tensors.
//
// Measured (bf16; bytes that have to move / kernel time): quantize 16384 x 11008 88 us, 6.2 TB/s; norm with residual
// 8192 x 4096 41 us, 5.7 TB/s; its backward pass 42 us + 4.5 us for the join of the partial sums, 6.4 TB/s; quantizing and
// restoring 16384 x 11008 together 171 us, 6.3 TB/s.

#include "int8_common.h"

namespace {

using namespace optimi_int8;

constexpr int kBlock = 256;         // lanes of a workgroup, or TEAM where that is more
constexpr int kWaveRowCols = 1024;  // rows up to here belong to one wavefront: no LDS, no barrier
constexpr int kLongCols = 16384;    // rows beyond do not stay in registers
template <int TEAM>
constexpr int kLanes = TEAM > kBlock ? TEAM : kBlock;

// Grids stay far below the 2^32 threads that a launch may have; a workgroup takes further rows in a loop.
constexpr int64_t kMaxBlocks = 1 << 20;
inline unsigned blocks_for(int64_t rows, int per_block) {
  const int64_t n = (rows + per_block - 1) / per_block;
  return (unsigned)(n < kMaxBlocks ? n : kMaxBlocks);
}

// A row of up to 8 * TEAM * VPT elements, vector v of lane l at element (v * TEAM + l) * 8.
template <int TEAM>
struct Place {
  int lane;     // in the team
  int64_t row;  // the team's first row
  int64_t step; // rows that the whole grid takes at once
  __device__ __forceinline__ Place() {
    lane = threadIdx.x % TEAM;
    row = (int64_t)blockIdx.x * (kLanes<TEAM> / TEAM) + __builtin_amdgcn_readfirstlane((int)threadIdx.x / TEAM);
    step = (int64_t)gridDim.x * (kLanes<TEAM> / TEAM);
  }
};

// The eight elements from c on of a row.  Where the row ends inside of them, the vector is the row's last eight elements: some
// of them are the neighbour's too, which computes and stores the same for them, so a row of any width takes whole
// vectors only, without a branch.  A row of less than eight elements (TINY) is the exception.
__device__ __forceinline__ int place8(int c, int cols) { return c + 8 <= cols ? c : cols - 8; }
template <int DT, bool TINY>
__device__ __forceinline__ typename Elem<DT>::Raw load8(const typename Elem<DT>::type* row, int c, int cols) {
  if (TINY && cols < 8) return load_some<DT>(row, cols);
  return Elem<DT>::load(row + place8(c, cols));
}
// The same for what is read once.
template <int DT, bool TINY>
__device__ __forceinline__ typename Elem<DT>::Raw stream8(const typename Elem<DT>::type* row, int c, int cols) {
  if (TINY && cols < 8) return load_some<DT>(row, cols);
  return Elem<DT>::stream(row + place8(c, cols));
}
template <int DT, bool TINY>
__device__ __forceinline__ void store8(typename Elem<DT>::type* row, int c, int cols, const float (&f)[8], bool stream = false) {
  if (TINY && cols < 8) store_some<DT>(row, f, cols);
  else if (stream) Elem<DT>::stream_out(row + place8(c, cols), Elem<DT>::pack(f));
  else Elem<DT>::store(row + place8(c, cols), Elem<DT>::pack(f));
}
template <bool TINY>
__device__ __forceinline__ void store_values8(int8_t* row, int c, int cols, u32x2 v) {
  if (TINY && cols < 8) store_values(row, v, cols);
  else store_values(row + place8(c, cols), v, 8);
}
// For sums: the elements that the neighbour has as well count once.
template <bool TINY>
__device__ __forceinline__ void once(float (&f)[8], int c, int cols) {
  if (cols % 8 == 0 || (TINY && cols < 8)) return;
  const int skip = c - place8(c, cols);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = i < skip ? 0.0f : f[i];
}

template <int DT, int TEAM, int VPT>
__global__ void __launch_bounds__(kLanes<TEAM>) quantize_kernel(const typename Elem<DT>::type* __restrict__ x, int64_t rows, int cols,
                                                          int8_t* __restrict__ values, float* __restrict__ scales) {
  using E = Elem<DT>;
  constexpr bool kTiny = TEAM == 64 && VPT == 1;
  __shared__ uint32_t slots[2][kLanes<TEAM> / 64];
  const Place<TEAM> at;
  // a team of several waves has the workgroup to itself, so all of its waves make the same number of rounds
  int turn = 0;
  for (int64_t row = at.row; row < rows; row += at.step, turn ^= 1) {
    const typename E::type* in = x + row * cols;
    typename E::Raw raw[VPT];
    uint32_t most = 0;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = (v * TEAM + at.lane) * 8;
      raw[v] = E::zero();
      if (c < cols) raw[v] = stream8<DT, kTiny>(in, c, cols);
    }
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      float f[8];
      E::unpack(raw[v], f);
#pragma unroll
      for (int i = 0; i < 8; ++i) most = MaxOp::join(most, abs_bits(f[i]));
    }
    most = team_reduce<MaxOp, TEAM>(most, slots[turn]);
    const RowScale s = row_scale<DT>(most);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = (v * TEAM + at.lane) * 8;
      float f[8];
      E::unpack(raw[v], f);
      if (c < cols) store_values8<kTiny>(values + row * cols, c, cols, quantize8(f, s));
    }
    if (at.lane == 0) scales[row] = s.scale;
  }
}

// Rows that do not fit the registers: one workgroup each, read twice.
template <int DT>
__global__ void __launch_bounds__(kBlock) quantize_long_kernel(const typename Elem<DT>::type* __restrict__ x, int64_t rows, int cols,
                                                               int8_t* __restrict__ values, float* __restrict__ scales) {
  using E = Elem<DT>;
  __shared__ uint32_t slots[2][kBlock / 64];
  int turn = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
    const typename E::type* in = x + row * cols;
    uint32_t most = 0;
    for (int c = threadIdx.x * 8; c < cols; c += kBlock * 8) {
      float f[8];
      E::unpack(load8<DT, false>(in, c, cols), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) most = MaxOp::join(most, abs_bits(f[i]));
    }
    most = team_reduce<MaxOp, kBlock>(most, slots[turn]);
    const RowScale s = row_scale<DT>(most);
    for (int c = threadIdx.x * 8; c < cols; c += kBlock * 8) {
      float f[8];
      E::unpack(load8<DT, false>(in, c, cols), f);
      store_values8<false>(values + row * cols, c, cols, quantize8(f, s));
    }
    if (threadIdx.x == 0) scales[row] = s.scale;
  }
}

// q * s, eight values a lane; `team` lanes (a power of two) share a row.
template <int DT>
__global__ void __launch_bounds__(kBlock) dequantize_kernel(const int8_t* __restrict__ values, const float* __restrict__ scales, int64_t rows,
                                                            int cols, int team, typename Elem<DT>::type* __restrict__ out) {
  const int lane = threadIdx.x % team;
  for (int64_t row = (int64_t)blockIdx.x * (kBlock / team) + threadIdx.x / team; row < rows; row += (int64_t)gridDim.x * (kBlock / team)) {
    const float s = scales[row];
    const int8_t* from = values + row * cols;
    for (int c = lane * 8; c < cols; c += team * 8) {
      float f[8];
      if (cols >= 8) {
        const u32x2 q = __builtin_nontemporal_load((const u32x2_align1*)(from + place8(c, cols)));
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)(int8_t)(q[i / 4] >> (8 * (i % 4))) * s;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)from[i < cols ? i : 0] * s;
      }
      store8<DT, true>(out + row * cols, c, cols, f, whole_lines(cols, sizeof(typename Elem<DT>::type)));
    }
  }
}

// The norm's weight in its own type: that of the activations or fp32.
template <int DT, bool W32>
struct Weight {
  static constexpr int kType = W32 ? (int)OPTIMI_F32 : DT;
  using E = Elem<kType>;
  template <bool TINY>
  static __device__ __forceinline__ void load(const void* w, int c, int cols, float (&f)[8]) {
    E::unpack(load8<kType, TINY>((const typename E::type*)w, c, cols), f);
  }
};

// h = x + residual, rounded to the type it is kept in; the norm is that of the kept values, which is what the
// backward pass will see.
template <int DT>
__device__ __forceinline__ typename Elem<DT>::Raw add_rows(const typename Elem<DT>::Raw& x, const typename Elem<DT>::Raw& r) {
  float a[8], b[8];
  Elem<DT>::unpack(x, a);
  Elem<DT>::unpack(r, b);
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] += b[i];
  return Elem<DT>::pack(a);
}

struct NormArgs {
  const void *x, *residual, *weight;
  int64_t rows;
  int cols;
  float eps, eps_up, eps_down;  // eps itself, and in units of scaled squares
  float least;                  // sums of squares below are formed again: 0 where eps is what counts then
  void* h;
  int8_t* values;
  float *scales, *rstd;
};

// Rows of finite numbers can have squares outside of fp32's range: beyond 2^64 the sum is infinite, below 2^-63 terms lose bits or
// vanish, which counts in sums below 2^-96 if eps is no larger.  Such a row is summed a second time, its numbers (and the root
// of eps) scaled by 2^96 or 2^-96, which bring rows of either kind, up to the widest, into the range.
constexpr float kScaleUp = 0x1p96f, kScaleDown = 0x1p-96f, kLeastSum = 0x1p-96f;
__device__ __forceinline__ bool in_range(float sum_of_squares, const NormArgs& a) { return sum_of_squares >= a.least && sum_of_squares < INFINITY; }
__device__ __forceinline__ float scale_of(float sum_of_squares) { return sum_of_squares < kLeastSum ? kScaleUp : kScaleDown; }
__device__ __forceinline__ float inverse_rms(float sum_of_squares, float scale, const NormArgs& a) {
  const float eps = scale == 1.0f ? a.eps : scale == kScaleUp ? a.eps_up : a.eps_down;
  return 1.0f / sqrtf(sum_of_squares / (float)a.cols + eps);
}

// Two vectors a lane: seven waves per SIMD, for which the compiler by itself takes a few registers too many.  (Rows summed again behind the
// others' path instead, in code of its own: 512 columns 77 us instead of 68, and 60 instead of 58 for 8192 x 4096 with the restore.)
template <int DT, bool W32, int TEAM, int VPT>
__global__ void __launch_bounds__(kLanes<TEAM>, VPT == 2 ? 7 : 1) norm_kernel(NormArgs a) {
  using E = Elem<DT>;
  using T = typename E::type;
  constexpr bool kTiny = TEAM == 64 && VPT == 1;
  __shared__ uint32_t slots[2][3][kLanes<TEAM> / 64];
  const Place<TEAM> at;
  const int cols = a.cols;
  int turn = 0;
  for (int64_t row = at.row; row < a.rows; row += at.step, turn ^= 1) {
    typename E::Raw raw[VPT];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = (v * TEAM + at.lane) * 8;
      raw[v] = E::zero();
      if (c < cols) raw[v] = stream8<DT, kTiny>((const T*)a.x + row * cols, c, cols);
    }
    if (a.residual) {
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        const int c = (v * TEAM + at.lane) * 8;
        if (c < cols) {
          raw[v] = add_rows<DT>(raw[v], stream8<DT, kTiny>((const T*)a.residual + row * cols, c, cols));
          float f[8];
          E::unpack(raw[v], f);
          store8<DT, kTiny>((T*)a.h + row * cols, c, cols, f);
        }
      }
    }
    float f[VPT][8];
#pragma unroll
    for (int v = 0; v < VPT; ++v) E::unpack(raw[v], f[v]);
    float scale = 1.0f, sum;
    for (int pass = 0;; ++pass) {  // one pass, or two for the whole team
      sum = 0.0f;
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        float g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = f[v][i];
        once<kTiny>(g, (v * TEAM + at.lane) * 8, cols);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(g[i], g[i], sum);
      }
      sum = __uint_as_float(team_reduce<SumOp, TEAM>(__float_as_uint(sum), slots[turn][pass]));
      if (pass > 0 || in_range(sum, a)) break;
      scale = scale_of(sum);
#pragma unroll
      for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) f[v][i] *= scale;
    }
    const float r = inverse_rms(sum, scale, a);  // of the scaled row
    uint32_t most = 0;
    float y[VPT][8];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = (v * TEAM + at.lane) * 8;
      float w[8];
      if (c < cols) {
        Weight<DT, W32>::template load<kTiny>(a.weight, c, cols, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[v][i] = f[v][i] * r * w[i];
          most = MaxOp::join(most, abs_bits(y[v][i]));
        }
      }
    }
    most = team_reduce<MaxOp, TEAM>(most, slots[turn][2]);
    const RowScale s = row_scale<OPTIMI_F32>(most);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = (v * TEAM + at.lane) * 8;
      if (c < cols) store_values8<kTiny>(a.values + row * cols, c, cols, quantize8(y[v], s));
    }
    if (at.lane == 0) {
      a.scales[row] = s.scale;
      a.rstd[row] = scale * r;
    }
  }
}

template <int DT, bool W32>
__global__ void __launch_bounds__(kBlock) norm_long_kernel(NormArgs a) {
  using E = Elem<DT>;
  using T = typename E::type;
  __shared__ uint32_t slots[2][3][kBlock / 64];
  const int cols = a.cols;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const T* x = (const T*)a.x + row * cols;
    const T* res = a.residual ? (const T*)a.residual + row * cols : nullptr;
    auto kept = [&](int c, float (&f)[8]) {  // h, formed again from its two terms wherever it is needed
      typename E::Raw raw = load8<DT, false>(x, c, cols);
      if (res) raw = add_rows<DT>(raw, load8<DT, false>(res, c, cols));
      E::unpack(raw, f);
    };
    float scale = 1.0f, sum;
    for (int pass = 0;; ++pass) {
      sum = 0.0f;
      for (int c = threadIdx.x * 8; c < cols; c += kBlock * 8) {
        float f[8];
        kept(c, f);
        once<false>(f, c, cols);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(f[i] * scale, f[i] * scale, sum);
      }
      sum = __uint_as_float(team_reduce<SumOp, kBlock>(__float_as_uint(sum), slots[turn][pass]));
      if (pass > 0 || in_range(sum, a)) break;
      scale = scale_of(sum);
    }
    const float r = inverse_rms(sum, scale, a);
    uint32_t most = 0;
    for (int c = threadIdx.x * 8; c < cols; c += kBlock * 8) {
      float f[8], w[8];
      kept(c, f);
      Weight<DT, W32>::template load<false>(a.weight, c, cols, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) most = MaxOp::join(most, abs_bits(f[i] * scale * r * w[i]));
    }
    most = team_reduce<MaxOp, kBlock>(most, slots[turn][2]);
    const RowScale s = row_scale<OPTIMI_F32>(most);
    for (int c = threadIdx.x * 8; c < cols; c += kBlock * 8) {
      float f[8], w[8], y[8];
      kept(c, f);
      Weight<DT, W32>::template load<false>(a.weight, c, cols, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = f[i] * scale * r * w[i];
      store_values8<false>(a.values + row * cols, c, cols, quantize8(y, s));
      if (res) store8<DT, false>((T*)a.h + row * cols, c, cols, f);
    }
    if (threadIdx.x == 0) {
      a.scales[row] = s.scale;
      a.rstd[row] = scale * r;
    }
  }
}

// Backward pass of y = h r w with r = (mean h^2 + eps)^(-1/2), g = dL/dy:
//   dL/dh_i = r (g_i w_i - xhat_i mean(g w xhat)),  xhat = h r,  plus what arrives on the residual path;
//   dL/dw_i = sum over rows of g_i xhat_i.
// The second sum runs over rows: each team adds up its own rows in registers, a workgroup leaves one partial row in the
// workspace, and a second launch adds the partial rows in a fixed order - no atomics, the same bits on every run.
struct NormBackwardArgs {
  const void *grad, *grad_h, *h, *weight;
  const float* rstd;
  int64_t rows;
  int cols;
  void* dx;
  float* partial;  // [workgroups][cols]
};

template <int DT, bool W32, int TEAM, int VPT>
__global__ void __launch_bounds__(kLanes<TEAM>) norm_backward_kernel(NormBackwardArgs a) {
  using E = Elem<DT>;
  using T = typename E::type;
  constexpr bool kTiny = TEAM == 64 && VPT == 1;
  __shared__ uint32_t slots[2][kLanes<TEAM> / 64];
  const Place<TEAM> at;
  const int cols = a.cols;
  float w[VPT][8], dw[VPT][8];
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int c = (v * TEAM + at.lane) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[v][i] = dw[v][i] = 0.0f;
    if (c < cols) Weight<DT, W32>::template load<kTiny>(a.weight, c, cols, w[v]);
  }
  int turn = 0;
  for (int64_t row = at.row; row < a.rows; row += at.step, turn ^= 1) {
    typename E::Raw g[VPT], h[VPT], more[VPT];
    const float r = a.rstd[row];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = (v * TEAM + at.lane) * 8;
      g[v] = h[v] = more[v] = E::zero();
      if (c < cols) {
        g[v] = stream8<DT, kTiny>((const T*)a.grad + row * cols, c, cols);
        h[v] = stream8<DT, kTiny>((const T*)a.h + row * cols, c, cols);
        if (a.grad_h) more[v] = stream8<DT, kTiny>((const T*)a.grad_h + row * cols, c, cols);
      }
    }
    float dot = 0.0f;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      float fg[8], fh[8];
      float gw[8];
      E::unpack(g[v], fg);
      E::unpack(h[v], fh);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        fh[i] *= r;
        dw[v][i] = fmaf(fg[i], fh[i], dw[v][i]);
        gw[i] = fg[i] * w[v][i];
      }
      once<kTiny>(gw, (v * TEAM + at.lane) * 8, cols);
#pragma unroll
      for (int i = 0; i < 8; ++i) dot = fmaf(gw[i], fh[i], dot);
    }
    dot = __uint_as_float(team_reduce<SumOp, TEAM>(__float_as_uint(dot), slots[turn]));
    const float mean = dot / (float)cols;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = (v * TEAM + at.lane) * 8;
      float fg[8], fh[8], fm[8], d[8];
      E::unpack(g[v], fg);
      E::unpack(h[v], fh);
      E::unpack(more[v], fm);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = fmaf(r, fg[i] * w[v][i] - fh[i] * r * mean, fm[i]);
      if (c < cols) store8<DT, kTiny>((T*)a.dx + row * cols, c, cols, d);
    }
  }
  if constexpr (TEAM > 64) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = (v * TEAM + at.lane) * 8;
      if (c < cols) store8<OPTIMI_F32, kTiny>(a.partial + (int64_t)blockIdx.x * cols, c, cols, dw[v]);
    }
  } else {  // the workgroup's four teams leave one row
    __shared__ float join[kBlock / 64][kWaveRowCols];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = (v * TEAM + at.lane) * 8;
      const int to = kTiny && cols < 8 ? 0 : place8(c, cols);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c < cols && to + i < cols) join[threadIdx.x / 64][to + i] = dw[v][i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += kBlock) a.partial[(int64_t)blockIdx.x * cols + c] = join[0][c] + join[1][c] + join[2][c] + join[3][c];
  }
}

template <int DT, bool W32>
__global__ void __launch_bounds__(kBlock) norm_backward_long_kernel(NormBackwardArgs a) {
  using E = Elem<DT>;
  using T = typename E::type;
  __shared__ uint32_t slots[2][kBlock / 64];
  const int cols = a.cols;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const T* grad = (const T*)a.grad + row * cols;
    const T* h = (const T*)a.h + row * cols;
    const float r = a.rstd[row];
    float dot = 0.0f;
    for (int c = threadIdx.x * 8; c < cols; c += kBlock * 8) {
      float fg[8], fh[8], w[8];
      E::unpack(load8<DT, false>(grad, c, cols), fg);
      E::unpack(load8<DT, false>(h, c, cols), fh);
      Weight<DT, W32>::template load<false>(a.weight, c, cols, w);
      once<false>(fg, c, cols);
#pragma unroll
      for (int i = 0; i < 8; ++i) dot = fmaf(fg[i] * w[i], fh[i] * r, dot);
    }
    dot = __uint_as_float(team_reduce<SumOp, kBlock>(__float_as_uint(dot), slots[turn]));
    const float mean = dot / (float)cols;
    for (int c = threadIdx.x * 8; c < cols; c += kBlock * 8) {
      float fg[8], fh[8], fm[8], w[8], d[8];
      E::unpack(load8<DT, false>(grad, c, cols), fg);
      E::unpack(load8<DT, false>(h, c, cols), fh);
      E::unpack(a.grad_h ? load8<DT, false>((const T*)a.grad_h + row * cols, c, cols) : E::zero(), fm);
      Weight<DT, W32>::template load<false>(a.weight, c, cols, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = fmaf(r, fg[i] * w[i] - fh[i] * r * mean, fm[i]);
      store8<DT, false>((T*)a.dx + row * cols, c, cols, d);
    }
  }
}

// Sums over rows of a stripe of columns: of x itself (NORM false), or of g h r (NORM true, the weight gradient of
// norms whose rows do not stay in registers).  blockIdx.x is the stripe of 8 * kBlock columns, blockIdx.y takes every
// gridDim.y-th row and leaves a partial row.
template <int DT, bool NORM>
__global__ void __launch_bounds__(kBlock) column_partial_kernel(const typename Elem<DT>::type* __restrict__ x, const typename Elem<DT>::type* __restrict__ h,
                                                                const float* __restrict__ rstd, int64_t rows, int cols, float* __restrict__ partial) {
  using E = Elem<DT>;
  const int c = (blockIdx.x * kBlock + threadIdx.x) * 8;
  if (c >= cols) return;
  float sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] = 0.0f;
#pragma unroll 4
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    float f[8];
    E::unpack(load8<DT, true>(x + row * cols, c, cols), f);
    if constexpr (NORM) {
      float fh[8];
      E::unpack(load8<DT, true>(h + row * cols, c, cols), fh);
      const float r = rstd[row];
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] = fmaf(f[i], fh[i] * r, sum[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += f[i];
    }
  }
  store8<OPTIMI_F32, true>(partial + (int64_t)blockIdx.y * cols, c, cols, sum);
}

// Adds the partial rows: 32 columns a workgroup, its groups of 32 lanes each take every kJoin-th partial row.
constexpr int kJoin = 32;  // as many groups as columns: see the end
template <int OUT>
__global__ void __launch_bounds__(32 * kJoin) column_finish_kernel(const float* __restrict__ partial, int64_t parts, int64_t cols,
                                                                   typename Elem<OUT>::type* __restrict__ out) {
  __shared__ float sums[kJoin][33];
  const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
  for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < cols; c0 += (int64_t)gridDim.x * 32) {
    float s = 0.0f;
    if (c0 + lane < cols) {
#pragma unroll 8
      for (int64_t p = group; p < parts; p += kJoin) s += partial[p * cols + c0 + lane];
    }
    sums[group][lane] = s;
    __syncthreads();
    float sum = sums[lane][group];  // a group of lanes for each of the 32 columns
#pragma unroll
    for (int d = 16; d > 0; d /= 2) sum += __shfl_xor(sum, d, 32);
    if (lane == 0 && c0 + group < cols) out[c0 + group] = Elem<OUT>::put(sum);
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------

// Calls f(team, vectors per lane) for rows of `cols` elements that stay in registers.
template <class F>
int by_width(int64_t cols, F f) {
#define OPTIMI_WIDTH(team, vpt) \
  if (cols <= (int64_t)8 * team * vpt) return f(std::integral_constant<int, team>{}, std::integral_constant<int, vpt>{})
  OPTIMI_WIDTH(64, 1);
  OPTIMI_WIDTH(64, 2);
  static_assert(kWaveRowCols == 64 * 8 * 2, "the widest row of one wavefront");
  OPTIMI_WIDTH(256, 1);
  OPTIMI_WIDTH(256, 2);
  OPTIMI_WIDTH(256, 3);
  OPTIMI_WIDTH(256, 4);
  OPTIMI_WIDTH(512, 3);
  static_assert(kLongCols == 512 * 8 * 4, "the widest row that stays in registers");
  return f(std::integral_constant<int, 512>{}, std::integral_constant<int, 4>{});
#undef OPTIMI_WIDTH
}

inline int rows_per_block(int64_t cols) { return cols <= kWaveRowCols ? kBlock / 64 : 1; }

// Workgroups of a pass that ends in partial rows: enough of them to fill the machine, few enough for the partial rows to be a
// small part of the traffic - four rows a team, but not below 128 workgroups.  (400 x 8256 bf16: 19.8 us with a workgroup
// for every row, 14.7 us with 128; 16384 x 1024: 28 us with four rows of partial sums per workgroup, 24 us with one.)
inline int64_t partial_blocks(int64_t rows, int64_t cols) {
  const int per = rows_per_block(cols);
  const int64_t most = (rows + per - 1) / per, four = (rows + 4 * per - 1) / (4 * per);
  const int64_t n = four > 512 ? 512 : four < 128 ? 128 : four;
  return n < most ? n : most;
}
inline int64_t norm_partials(int64_t rows, int64_t cols) {
  if (cols > kLongCols) return rows < 64 ? rows : 64;
  return partial_blocks(rows, cols);
}

}  // namespace

namespace optimi_int8 {

int finish_columns(const float* partial, int64_t parts, int64_t cols, int dtype, void* out, hipStream_t stream) {
  if (cols == 0) return 0;
  return by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    column_finish_kernel<DT><<<dim3(blocks_for(cols, 32)), dim3(32 * kJoin), 0, stream>>>(partial, parts, cols, (typename Elem<DT>::type*)out);
    OPTIMI_INT8_TRY(hipGetLastError());
    return 0;
  });
}

// Column sums of a [rows, cols] matrix, for bias gradients: see int8_gemm.hip.
int64_t column_sum_workspace(int64_t rows, int64_t cols) { return (rows < 128 ? rows : 128) * cols * 4; }

int column_sum(const void* x, int64_t rows, int64_t cols, int dtype, void* out, void* workspace, hipStream_t stream) {
  if (cols == 0) return 0;
  const int64_t parts = rows < 128 ? rows : 128;
  return by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    using T = typename Elem<DT>::type;
    const unsigned stripes = (unsigned)((cols + kBlock * 8 - 1) / (kBlock * 8));
    if (parts > 0) {
      column_partial_kernel<DT, false><<<dim3(stripes, (unsigned)parts), dim3(kBlock), 0, stream>>>((const T*)x, nullptr, nullptr, rows, (int)cols, (float*)workspace);
      OPTIMI_INT8_TRY(hipGetLastError());
    }
    return finish_columns((const float*)workspace, parts, cols, dtype, out, stream);
  });
}

}  // namespace optimi_int8

extern "C" {

int optimi_hip_int8_quantize(const void* x, int64_t rows, int64_t cols, int dtype, int8_t* values, float* scales, optimi_stream_t stream_) {
  if (!valid_dtype(dtype)) return OPTIMI_ERR_DTYPE;
  if (int rc = check_shape(rows, cols)) return rc;
  if (rows == 0) return 0;
  if (!scales || (cols && (!x || !values))) return OPTIMI_ERR_NULL;
  if (!aligned_to(x, elem_bytes(dtype)) || !aligned_to(scales, 4)) return OPTIMI_ERR_ALIGN;
  hipStream_t stream = (hipStream_t)stream_;
  return by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    using T = typename Elem<DT>::type;
    if (cols > kLongCols) {
      quantize_long_kernel<DT><<<dim3(blocks_for(rows, 1)), dim3(kBlock), 0, stream>>>((const T*)x, rows, (int)cols, values, scales);
    } else {
      by_width(cols, [&](auto team, auto vpt) {
        quantize_kernel<DT, decltype(team)::value, decltype(vpt)::value>
            <<<dim3(blocks_for(rows, rows_per_block(cols))), dim3(kLanes<decltype(team)::value>), 0, stream>>>((const T*)x, rows, (int)cols, values, scales);
        return 0;
      });
    }
    OPTIMI_INT8_TRY(hipGetLastError());
    return 0;
  });
}

int optimi_hip_int8_dequantize(const int8_t* values, const float* scales, int64_t rows, int64_t cols, int dtype, void* out, optimi_stream_t stream_) {
  if (!valid_dtype(dtype)) return OPTIMI_ERR_DTYPE;
  if (int rc = check_shape(rows, cols)) return rc;
  if (rows == 0 || cols == 0) return 0;
  if (!values || !scales || !out) return OPTIMI_ERR_NULL;
  if (!aligned_to(out, elem_bytes(dtype)) || !aligned_to(scales, 4)) return OPTIMI_ERR_ALIGN;
  int team = 1;
  while (team < kBlock && (int64_t)team * 8 < cols) team *= 2;
  return by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    dequantize_kernel<DT><<<dim3(blocks_for(rows, kBlock / team)), dim3(kBlock), 0, (hipStream_t)stream_>>>(values, scales, rows, (int)cols, team,
                                                                                                         (typename Elem<DT>::type*)out);
    OPTIMI_INT8_TRY(hipGetLastError());
    return 0;
  });
}

int optimi_hip_add_rms_norm_int8(const void* x, const void* residual, const void* weight, int64_t rows, int64_t cols, int dtype, int weight_dtype,
                                 double eps, void* h, int8_t* values, float* scales, float* rstd, optimi_stream_t stream_) {
  if (!valid_dtype(dtype) || (weight_dtype != dtype && weight_dtype != OPTIMI_F32)) return OPTIMI_ERR_DTYPE;
  if (int rc = check_shape(rows, cols)) return rc;
  if (!(eps >= 0.0)) return OPTIMI_ERR_ARG;
  if (rows == 0) return 0;
  if (cols == 0) return OPTIMI_ERR_SIZE;  // the mean of no elements
  if (!x || !weight || !values || !scales || !rstd || (residual && !h)) return OPTIMI_ERR_NULL;
  const int64_t size = elem_bytes(dtype);
  if (!aligned_to(x, size) || !aligned_to(residual, size) || !aligned_to(h, size) || !aligned_to(weight, elem_bytes(weight_dtype)) ||
      !aligned_to(scales, 4) || !aligned_to(rstd, 4))
    return OPTIMI_ERR_ALIGN;
  hipStream_t stream = (hipStream_t)stream_;
  const double up = (double)kScaleUp * kScaleUp, down = (double)kScaleDown * kScaleDown;
  const NormArgs args{x, residual, weight, rows, (int)cols, (float)eps, (float)(eps * up), (float)(eps * down), eps < kLeastSum ? kLeastSum : 0.0f, h, values, scales, rstd};
  return by_dtype(dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    auto with = [&](auto w32) {
      constexpr bool W32 = decltype(w32)::value;
      if (cols > kLongCols) {
        norm_long_kernel<DT, W32><<<dim3(blocks_for(rows, 1)), dim3(kBlock), 0, stream>>>(args);
      } else {
        by_width(cols, [&](auto team, auto vpt) {
          norm_kernel<DT, W32, decltype(team)::value, decltype(vpt)::value><<<dim3(blocks_for(rows, rows_per_block(cols))), dim3(kLanes<decltype(team)::value>), 0, stream>>>(args);
          return 0;
        });
      }
      OPTIMI_INT8_TRY(hipGetLastError());
      return 0;
    };
    if (weight_dtype == dtype) return with(std::false_type{});
    return with(std::true_type{});
  });
}

int64_t optimi_hip_add_rms_norm_int8_backward_workspace(int64_t rows, int64_t cols) {
  if (int rc = check_shape(rows, cols)) return rc;
  if (cols == 0) return OPTIMI_ERR_SIZE;
  return norm_partials(rows, cols) * cols * 4;
}

int optimi_hip_add_rms_norm_int8_backward(const void* grad, const void* grad_h, const void* h, const float* rstd, const void* weight, int64_t rows,
                                          int64_t cols, int dtype, int weight_dtype, void* dx, void* dweight, void* workspace, optimi_stream_t stream_) {
  if (!valid_dtype(dtype) || (weight_dtype != dtype && weight_dtype != OPTIMI_F32)) return OPTIMI_ERR_DTYPE;
  if (int rc = check_shape(rows, cols)) return rc;
  if (cols == 0) return OPTIMI_ERR_SIZE;
  if (!weight || !dweight || (rows && (!grad || !h || !rstd || !dx || !workspace))) return OPTIMI_ERR_NULL;
  const int64_t size = elem_bytes(dtype), wsize = elem_bytes(weight_dtype);
  if (!aligned_to(grad, size) || !aligned_to(grad_h, size) || !aligned_to(h, size) || !aligned_to(dx, size) || !aligned_to(weight, wsize) ||
      !aligned_to(dweight, wsize) || !aligned_to(rstd, 4) || !aligned_to(workspace, 4))
    return OPTIMI_ERR_ALIGN;
  hipStream_t stream = (hipStream_t)stream_;
  const int64_t parts = norm_partials(rows, cols);
  if (rows > 0) {
    const NormBackwardArgs args{grad, grad_h, h, weight, rstd, rows, (int)cols, dx, (float*)workspace};
    const int rc = by_dtype(dtype, [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      using T = typename Elem<DT>::type;
      auto with = [&](auto w32) {
        constexpr bool W32 = decltype(w32)::value;
        if (cols > kLongCols) {
          norm_backward_long_kernel<DT, W32><<<dim3(blocks_for(rows, 1)), dim3(kBlock), 0, stream>>>(args);
          OPTIMI_INT8_TRY(hipGetLastError());
          const unsigned stripes = (unsigned)((cols + kBlock * 8 - 1) / (kBlock * 8));
          column_partial_kernel<DT, true><<<dim3(stripes, (unsigned)parts), dim3(kBlock), 0, stream>>>((const T*)grad, (const T*)h, rstd, rows, (int)cols, (float*)workspace);
        } else {
          by_width(cols, [&](auto team, auto vpt) {
            norm_backward_kernel<DT, W32, decltype(team)::value, decltype(vpt)::value>
                <<<dim3((unsigned)partial_blocks(rows, cols)), dim3(kLanes<decltype(team)::value>), 0, stream>>>(args);
            return 0;
          });
        }
        OPTIMI_INT8_TRY(hipGetLastError());
        return 0;
      };
      if (weight_dtype == dtype) return with(std::false_type{});
      return with(std::true_type{});
    });
    if (rc) return rc;
  }
  return finish_columns((const float*)workspace, parts, cols, weight_dtype, dweight, stream);
}

}  // extern "C"
