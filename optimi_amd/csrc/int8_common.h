// What the int8 activation kernels share: element types, vector loads and stores that need no more than
// element alignment, reductions over the lanes that work on one row, and the row scale.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "optimi_hip.h"

namespace optimi_int8 {

#define OPTIMI_INT8_TRY(expr)                   \
  do {                                          \
    hipError_t err__ = (expr);                  \
    if (err__ != hipSuccess) return (int)err__; \
  } while (0)

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

inline bool valid_dtype(int dtype) { return dtype == OPTIMI_F32 || dtype == OPTIMI_BF16 || dtype == OPTIMI_F16; }
inline int64_t elem_bytes(int dtype) { return dtype == OPTIMI_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, int64_t bytes) { return ((uintptr_t)p % (uintptr_t)bytes) == 0; }

// Eight consecutive elements as they lie in memory, and as floats.  The loads and stores are written for
// addresses that are aligned to one element only: rows of an odd width start anywhere, gfx950 takes one
// 16-byte access at any such address, and an aligned one loses nothing by it.  stream and stream_out are for data that has
// left the caches before it is used again: what a row kernel reads once, and results larger than a cache, which
// would push out what is still needed (int8 product 8192 x 11008 x 4096: 359 us with ordinary stores, 341 us with these;
// restoring 16384 x 11008 values and quantizing them before: 201 us, 171 us).  Lines that two rows share must not be
// streamed out: they would be written in parts (fp32 weight gradient 4096 x 1023: 43 us, 53 us), hence whole_lines.
// (Where both kinds of a store stand in two branches, empty assembly keeps them apart: merged, they would lose the hint.)
__host__ __device__ inline bool whole_lines(int64_t cols, int size) { return cols * size % 64 == 0; }

template <int DT>
struct Elem;

template <>
struct Elem<OPTIMI_F32> {
  typedef float type;
  typedef u32x4 vec __attribute__((aligned(4)));
  struct Raw {
    u32x4 a, b;
  };
  static __device__ __forceinline__ float get(type v) { return v; }
  static __device__ __forceinline__ type put(float v) { return v; }
  static __device__ __forceinline__ Raw load(const type* p) { return {*(const vec*)p, *(const vec*)(p + 4)}; }
  static __device__ __forceinline__ Raw stream(const type* p) { return {__builtin_nontemporal_load((const vec*)p), __builtin_nontemporal_load((const vec*)(p + 4))}; }
  static __device__ __forceinline__ void store(type* p, const Raw& r) {
    *(vec*)p = r.a;
    *(vec*)(p + 4) = r.b;
  }
  static __device__ __forceinline__ void stream_out(type* p, const Raw& r) {
    asm volatile("");
    __builtin_nontemporal_store(r.a, (vec*)p);
    __builtin_nontemporal_store(r.b, (vec*)(p + 4));
    asm volatile("");
  }
  static __device__ __forceinline__ Raw zero() { return {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}}; }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = __uint_as_float(r.a[i]);
      f[4 + i] = __uint_as_float(r.b[i]);
    }
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[8]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.a[i] = __float_as_uint(f[i]);
      r.b[i] = __float_as_uint(f[4 + i]);
    }
    return r;
  }
};

struct Raw16 {
  u32x4 a;
};
typedef u32x4 u32x4_align2 __attribute__((aligned(2)));

template <>
struct Elem<OPTIMI_BF16> {
  typedef __bf16 type;
  typedef Raw16 Raw;
  static __device__ __forceinline__ float get(type v) { return (float)v; }
  static __device__ __forceinline__ type put(float v) { return (type)v; }
  static __device__ __forceinline__ Raw load(const type* p) { return {*(const u32x4_align2*)p}; }
  static __device__ __forceinline__ Raw stream(const type* p) { return {__builtin_nontemporal_load((const u32x4_align2*)p)}; }
  static __device__ __forceinline__ void store(type* p, const Raw& r) { *(u32x4_align2*)p = r.a; }
  static __device__ __forceinline__ void stream_out(type* p, const Raw& r) {
    asm volatile("");
    __builtin_nontemporal_store(r.a, (u32x4_align2*)p);
    asm volatile("");
  }
  static __device__ __forceinline__ Raw zero() { return {u32x4{0, 0, 0, 0}}; }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(r.a[i] << 16);
      f[2 * i + 1] = __uint_as_float(r.a[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[8]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.a[i] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)f[2 * i], (__bf16)f[2 * i + 1]});
    return r;
  }
};

template <>
struct Elem<OPTIMI_F16> {
  typedef _Float16 type;
  typedef Raw16 Raw;
  static __device__ __forceinline__ float get(type v) { return (float)v; }
  static __device__ __forceinline__ type put(float v) { return (type)v; }
  static __device__ __forceinline__ Raw load(const type* p) { return {*(const u32x4_align2*)p}; }
  static __device__ __forceinline__ Raw stream(const type* p) { return {__builtin_nontemporal_load((const u32x4_align2*)p)}; }
  static __device__ __forceinline__ void store(type* p, const Raw& r) { *(u32x4_align2*)p = r.a; }
  static __device__ __forceinline__ void stream_out(type* p, const Raw& r) {
    asm volatile("");
    __builtin_nontemporal_store(r.a, (u32x4_align2*)p);
    asm volatile("");
  }
  static __device__ __forceinline__ Raw zero() { return {u32x4{0, 0, 0, 0}}; }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t bits = r.a[i];  // a copy: the cast of a vector's element would take the first one
      const f16x2 h = __builtin_bit_cast(f16x2, bits);
      f[2 * i] = (float)h[0];
      f[2 * i + 1] = (float)h[1];
    }
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[8]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.a[i] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)f[2 * i], (_Float16)f[2 * i + 1]});
    return r;
  }
};

// Up to eight elements at the end of a row: `n` >= 1 of them exist, the others read as zero and are not written.  (The last
// one is loaded again in their place, so that all loads are in flight at once; a branch around each would wait for each.)
template <int DT>
__device__ __forceinline__ typename Elem<DT>::Raw load_some(const typename Elem<DT>::type* p, int64_t n) {
  if (n >= 8) return Elem<DT>::load(p);
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = Elem<DT>::get(p[i < n ? i : (int)n - 1]);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = i < n ? f[i] : 0.0f;
  return Elem<DT>::pack(f);
}
template <int DT>
__device__ __forceinline__ void store_some(typename Elem<DT>::type* p, const float (&f)[8], int64_t n, bool stream = false) {
  if (n >= 8) {
    if (stream) Elem<DT>::stream_out(p, Elem<DT>::pack(f));
    else Elem<DT>::store(p, Elem<DT>::pack(f));
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = Elem<DT>::put(f[i]);
}

typedef u32x2 u32x2_align1 __attribute__((aligned(1)));
typedef u32x4 u32x4_align1 __attribute__((aligned(1)));
__device__ __forceinline__ void store_values(int8_t* p, u32x2 v, int64_t n) {
  if (n >= 8) {
    *(u32x2_align1*)p = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = (int8_t)(v[i / 4] >> (8 * (i % 4)));
}

// Reductions over a wavefront without LDS traffic: four shifts inside the rows of 16 lanes, two broadcasts
// between them; lane 63 then holds the result.  Lanes that a shift leaves without a partner combine with 0,
// which is neutral for the sums and for the maxima (of bits of absolute values) taken here.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_or_zero(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
struct SumOp {
  static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }
};
struct MaxOp {
  static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b) { return a > b ? a : b; }
};
template <class Op>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t v) {
  v = Op::join(v, dpp_or_zero<0x111, 0xf>(v));  // row_shr:1
  v = Op::join(v, dpp_or_zero<0x112, 0xf>(v));  // row_shr:2
  v = Op::join(v, dpp_or_zero<0x114, 0xf>(v));  // row_shr:4
  v = Op::join(v, dpp_or_zero<0x118, 0xf>(v));  // row_shr:8
  v = Op::join(v, dpp_or_zero<0x142, 0xa>(v));  // row_bcast:15
  v = Op::join(v, dpp_or_zero<0x143, 0xc>(v));  // row_bcast:31
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// The same over the TEAM lanes that share a row.  `slots` is LDS of TEAM / 64 words that no other reduction of
// this row uses; a team of one wavefront needs none.  Every wave of the workgroup has to reach the call.
template <class Op, int TEAM>
__device__ __forceinline__ uint32_t team_reduce(uint32_t v, uint32_t* slots) {
  v = wave_reduce<Op>(v);
  if constexpr (TEAM > 64) {
    constexpr int kWaves = TEAM / 64;
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x / 64] = v;
    __syncthreads();
    v = slots[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v = Op::join(v, slots[w]);
  }
  return v;
}

// The scale of a row whose largest absolute value has the bits `absmax` (of a float): the smallest power of two
// s with absmax <= 127 s.  A power of two costs up to one bit against absmax / 127, and buys that x / s, q s and
// the products of scales are exact: a row means the same in every type and in every kernel that reads it, and no
// rounding but the one to a whole number is ever made.  Zero rows get 1; rows that hold an infinity or a NaN get
// NaN (and zeros), so that what is computed from them is NaN and an overflow is seen by whoever looks for one.
struct RowScale {
  float scale, inverse, limit;
  uint32_t mask;  // 0 for rows that are not finite: their values are zeros
};
template <int DT>
__device__ __forceinline__ RowScale row_scale(uint32_t absmax) {
  RowScale r;
  int e = (int)(absmax >> 23) - 6 + ((absmax & 0x7fffffu) > 0x7e0000u ? 1 : 0);  // biased; 127 = 1.984375 * 2^6
  if (e < 1) e = 1;  // scales are normal numbers
  if (absmax == 0) e = 127;
  r.scale = __uint_as_float((uint32_t)e << 23);
  r.inverse = __uint_as_float((uint32_t)(254 - e) << 23);
  // 64 steps of the largest scales lie beyond the type's range: values stay at 63 there, so that what they stand
  // for is finite in the type that the activation came from
  const int top = DT == OPTIMI_F16 ? 127 + 10 : 127 + 122;
  r.limit = e >= top ? 63.0f : 127.0f;
  r.mask = 0xffffffffu;
  if (absmax >= 0x7f800000u) {
    r.scale = __uint_as_float(0x7fc00000u);
    r.inverse = 0.0f;
    r.mask = 0u;
  }
  return r;
}

// rint(x / s) of eight values, ties to even, as int8.  x / s is exact, and adding 1.5 * 2^23 rounds it to a whole
// number whose low byte is the two's complement that is wanted.
__device__ __forceinline__ u32x2 quantize8(const float (&f)[8], const RowScale& r) {
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = __builtin_amdgcn_fmed3f(f[i] * r.inverse, -r.limit, r.limit);
    b[i] = __float_as_uint(q + 12582912.0f);
  }
  u32x2 v;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __builtin_amdgcn_perm(b[4 * i + 1], b[4 * i], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(b[4 * i + 3], b[4 * i + 2], 0x04000c0cu);
    v[i] = (lo | hi) & r.mask;
  }
  return v;
}

__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }

// Calls f with the dtype code as a type, for a code that was checked.
template <class F>
int by_dtype(int dtype, F f) {
  switch (dtype) {
    case OPTIMI_F32: return f(std::integral_constant<int, OPTIMI_F32>{});
    case OPTIMI_BF16: return f(std::integral_constant<int, OPTIMI_BF16>{});
    default: return f(std::integral_constant<int, OPTIMI_F16>{});
  }
}

// Grids are sized for rows below 2^31 and widths up to 2^28.
inline int check_shape(int64_t rows, int64_t cols) {
  return rows < 0 || cols < 0 || rows >= ((int64_t)1 << 31) || cols > ((int64_t)1 << 28) ? (int)OPTIMI_ERR_SIZE : 0;
}

// Column sums of a [rows, cols] matrix in its own type (int8_rows.hip); the workspace holds fp32 partial rows.
int finish_columns(const float* partial, int64_t parts, int64_t cols, int dtype, void* out, hipStream_t stream);  // the partial rows alone
int64_t column_sum_workspace(int64_t rows, int64_t cols);
int column_sum(const void* x, int64_t rows, int64_t cols, int dtype, void* out, void* workspace, hipStream_t stream);

}  // namespace optimi_int8
