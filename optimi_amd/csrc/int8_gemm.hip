// Matrix products of the int8 activations for MI355X (gfx950): the int8 product with scales per row and channel,
// and the weight gradient taken from an int8 checkpoint.

#include "int8_common.h"

namespace {

using namespace optimi_int8;

constexpr int kThreads = 256;
constexpr int kTile = 64;

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
};

// 16 bytes of a row from byte k on; what lies behind the row's end reads as zero.
__device__ __forceinline__ u32x4 load_bytes(const int8_t* row, int64_t k, int64_t len) {
  if (k + 16 <= len) return *(const u32x4_align1*)(row + k);
  u32x4 v{0, 0, 0, 0};
  for (int i = 0; i < 16 && k + i < len; ++i) v[i / 4] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i % 4));
  return v;
}

template <int DT>
__global__ void __launch_bounds__(kThreads) matmul_kernel(MatmulArgs p) {
  constexpr int kStep = 64, kPitch = kStep + 16;
  __shared__ __attribute__((aligned(16))) int8_t as[kTile * kPitch], bs[kTile * kPitch];
  const int64_t m0 = (int64_t)blockIdx.y * kTile, n0 = (int64_t)blockIdx.x * kTile;
  const int t = threadIdx.x, wave = t / 64, lane = t % 64;
  const int r = t / 4, c = (t % 4) * 16;
  const int wm = (wave / 2) * 32, wn = (wave % 2) * 32;
  i32x4 acc[2][2] = {};
  for (int64_t k0 = 0; k0 < p.k; k0 += kStep) {
    const u32x4 av = m0 + r < p.m ? load_bytes(p.a + (m0 + r) * p.k, k0 + c, p.k) : u32x4{0, 0, 0, 0};
    const u32x4 bv = n0 + r < p.n ? load_bytes(p.b + (n0 + r) * p.k, k0 + c, p.k) : u32x4{0, 0, 0, 0};
    __syncthreads();
    *(u32x4*)(as + r * kPitch + c) = av;
    *(u32x4*)(bs + r * kPitch + c) = bv;
    __syncthreads();
    i32x4 fa[2], fb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fa[i] = *(const i32x4*)(as + (wm + i * 16 + lane % 16) * kPitch + (lane / 16) * 16);
      fb[i] = *(const i32x4*)(bs + (wn + i * 16 + lane % 16) * kPitch + (lane / 16) * 16);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[i], fb[j], acc[i][j], 0, 0, 0);
  }
  using E = Elem<DT>;
  using T = typename E::type;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t n = n0 + wn + j * 16 + lane % 16;
    if (n >= p.n) continue;
    const float sb = p.b_scales[n], bias = p.bias ? E::get(((const T*)p.bias)[n]) : 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t m = m0 + wm + i * 16 + (lane / 16) * 4 + e;
        if (m < p.m) ((T*)p.out)[m * p.n + n] = E::put(fmaf((float)acc[i][j][e] * p.a_scales[m], sb, bias));
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
};

template <int DT>
struct Product;
template <>
struct Product<OPTIMI_BF16> {
  static constexpr int kPieces = 1;
  typedef __bf16 type;
  typedef bf16x8 frag;
  static __device__ __forceinline__ f32x4 mfma(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Product<OPTIMI_F16> {
  static constexpr int kPieces = 1;
  typedef _Float16 type;
  typedef f16x8 frag;
  static __device__ __forceinline__ f32x4 mfma(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Product<OPTIMI_F32> : Product<OPTIMI_BF16> {
  static constexpr int kPieces = 3;
};

// An fp32 number as the sum of three bf16 numbers, exactly: the upper 8 bits of what is left, three times.
__device__ __forceinline__ void split3(float x, __bf16 (&p)[3]) {
  if (abs_bits(x) >= 0x7f800000u) {
    p[0] = (__bf16)x;
    p[1] = p[2] = (__bf16)0.0f;
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const float top = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
    p[i] = (__bf16)top;
    x -= top;
  }
}

template <int DT>
__global__ void __launch_bounds__(kThreads) weight_grad_kernel(WeightGradArgs p) {
  using E = Elem<DT>;
  using T = typename E::type;
  using P = Product<DT>;
  using H = typename P::type;
  constexpr int kStep = 32, kPitch = kStep + 8;
  __shared__ __attribute__((aligned(16))) H as[P::kPieces][kTile * kPitch], bs[kTile * kPitch];
  const int64_t n0 = (int64_t)blockIdx.y * kTile, c0 = (int64_t)blockIdx.x * kTile;
  const int t = threadIdx.x, wave = t / 64, lane = t % 64;
  const int r = t / 8, c = (t % 8) * 8;
  const int wn = (wave / 2) * 32, wc = (wave % 2) * 32;
  f32x4 acc[2][2] = {};
  for (int64_t m0 = 0; m0 < p.rows; m0 += kStep) {
    const int64_t m = m0 + r;
    float g[8], q[8], s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = q[i] = 0.0f;
    if (m < p.rows) {
      s = p.scales[m];
      if (n0 + c < p.outs) E::unpack(load_some<DT>((const T*)p.grad + m * p.outs + n0 + c, p.outs - n0 - c), g);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + c + i < p.cols) q[i] = (float)p.values[m * p.cols + c0 + c + i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (P::kPieces == 1) {
        as[0][(c + i) * kPitch + r] = (H)g[i];
        bs[(c + i) * kPitch + r] = (H)(q[i] * s);
      } else {
        __bf16 pieces[3];
        split3(g[i] * s, pieces);
#pragma unroll
        for (int z = 0; z < 3; ++z) as[z][(c + i) * kPitch + r] = pieces[z];
        bs[(c + i) * kPitch + r] = (H)q[i];
      }
    }
    __syncthreads();
    typename P::frag fb[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) fb[j] = *(const typename P::frag*)(bs + (wc + j * 16 + lane % 16) * kPitch + (lane / 16) * 8);
#pragma unroll
    for (int z = P::kPieces - 1; z >= 0; --z)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const typename P::frag fa = *(const typename P::frag*)(as[z] + (wn + i * 16 + lane % 16) * kPitch + (lane / 16) * 8);
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = P::mfma(fa, fb[j], acc[i][j]);
      }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t k = c0 + wc + j * 16 + lane % 16;
    if (k >= p.cols) continue;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t n = n0 + wn + i * 16 + (lane / 16) * 4 + e;
        if (n < p.outs) ((T*)p.out)[n * p.cols + k] = E::put(acc[i][j][e]);
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

constexpr int64_t kMostSum = 131071;  // (-128)^2 times this stays below 2^31
constexpr int64_t kMostTiles = 65535;

}  // namespace

extern "C" {

int64_t optimi_hip_int8_matmul_workspace(int64_t m, int64_t n, int64_t k) {
  if (int rc = check_shape(m, n)) return rc;
  if (k < 0 || k > kMostSum) return OPTIMI_ERR_SIZE;
  return 0;
}

int optimi_hip_int8_matmul(const int8_t* a, const float* a_scales, const int8_t* b, const float* b_scales, const void* bias, int64_t m, int64_t n,
                           int64_t k, int dtype, void* out, void* workspace, optimi_stream_t stream) {
  (void)workspace;
  if (!valid_dtype(dtype)) return OPTIMI_ERR_DTYPE;
  if (int rc = check_shape(m, n)) return rc;
  if (k < 0 || k > kMostSum) return OPTIMI_ERR_SIZE;
  if (m == 0 || n == 0) return 0;
  if (!a_scales || !b_scales || !out || (k && (!a || !b))) return OPTIMI_ERR_NULL;
  const int64_t size = elem_bytes(dtype);
  if (!aligned_to(a_scales, 4) || !aligned_to(b_scales, 4) || !aligned_to(bias, size) || !aligned_to(out, size)) return OPTIMI_ERR_ALIGN;
  const int64_t tm = (m + kTile - 1) / kTile, tn = (n + kTile - 1) / kTile;
  if (tm > kMostTiles) return OPTIMI_ERR_SIZE;
  const MatmulArgs args{a, a_scales, b, b_scales, bias, m, n, k, out};
  return by_dtype(dtype, [&](auto dt) {
    matmul_kernel<decltype(dt)::value><<<dim3((unsigned)tn, (unsigned)tm), dim3(kThreads), 0, (hipStream_t)stream>>>(args);
    OPTIMI_INT8_TRY(hipGetLastError());
    return 0;
  });
}

int64_t optimi_hip_int8_weight_grad_workspace(int64_t rows, int64_t outs, int64_t cols, int dtype, int with_bias) {
  if (!valid_dtype(dtype)) return OPTIMI_ERR_DTYPE;
  if (int rc = check_shape(rows, outs)) return rc;
  if (int rc = check_shape(rows, cols)) return rc;
  return with_bias ? column_sum_workspace(rows, outs) : 0;
}

int optimi_hip_int8_weight_grad(const void* grad, const int8_t* values, const float* scales, int64_t rows, int64_t outs, int64_t cols, int dtype,
                                void* weight_grad, void* bias_grad, void* workspace, optimi_stream_t stream) {
  if (!valid_dtype(dtype)) return OPTIMI_ERR_DTYPE;
  if (int rc = check_shape(rows, outs)) return rc;
  if (int rc = check_shape(rows, cols)) return rc;
  if (outs == 0) return 0;
  if ((cols && !weight_grad) || (rows && (!grad || !scales || (cols && !values))) || (rows && bias_grad && !workspace)) return OPTIMI_ERR_NULL;
  const int64_t size = elem_bytes(dtype);
  if (!aligned_to(grad, size) || !aligned_to(scales, 4) || !aligned_to(weight_grad, size) || !aligned_to(bias_grad, size) || !aligned_to(workspace, 4))
    return OPTIMI_ERR_ALIGN;
  if (bias_grad) {
    if (int rc = column_sum(grad, rows, outs, dtype, bias_grad, workspace, (hipStream_t)stream)) return rc;
  }
  if (cols == 0) return 0;
  const int64_t tn = (outs + kTile - 1) / kTile, tc = (cols + kTile - 1) / kTile;
  if (tn > kMostTiles) return OPTIMI_ERR_SIZE;
  const WeightGradArgs args{grad, values, scales, rows, outs, cols, weight_grad};
  return by_dtype(dtype, [&](auto dt) {
    weight_grad_kernel<decltype(dt)::value><<<dim3((unsigned)tc, (unsigned)tn), dim3(kThreads), 0, (hipStream_t)stream>>>(args);
    OPTIMI_INT8_TRY(hipGetLastError());
    return 0;
  });
}

}  // extern "C"
