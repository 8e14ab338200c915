// Shared by the kernels of the network in front of the determinants (relative position bias,
// attention, its step over a paged cache, residual norms): element types, vector loads, wave
// sums, distance buckets.
#pragma once
#include "common.h"
#include "fermix_internal.h"

namespace fx {
namespace net {

template <class T, int V>
using vec_t = T __attribute__((ext_vector_type(V)));

template <class T>
__device__ __forceinline__ float to_f32(T x) {
  return (float)x;
}

// Elements of a 16-byte vector.
template <class T>
constexpr int VEC16 = 16 / (int)sizeof(T);

template <int CTRL>
__device__ __forceinline__ float dpp_f32(float x) {
  return __uint_as_float(dpp_u32<CTRL>(__float_as_uint(x)));
}

struct AddOp {
  static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct MaxOp {
  static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};

// x joined with that of the lane 16 or 32 away.
template <class OP>
__device__ __forceinline__ float join16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return OP::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <class OP>
__device__ __forceinline__ float join32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return OP::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Sum over the aligned group of W lanes (W a power of two up to 64); every lane gets it. No LDS: quad
// permutes, mirrors, then swaps of rows.
template <int W>
__device__ __forceinline__ float group_sum(float x) {
  if constexpr (W >= 2) x += dpp_f32<0xB1>(x);   // quad_perm [1,0,3,2]
  if constexpr (W >= 4) x += dpp_f32<0x4E>(x);   // quad_perm [2,3,0,1]
  if constexpr (W >= 8) x += dpp_f32<0x141>(x);  // row_half_mirror
  if constexpr (W >= 16) x += dpp_f32<0x140>(x); // row_mirror
  if constexpr (W >= 32) x = join16<AddOp>(x);
  if constexpr (W >= 64) x = join32<AddOp>(x);
  return x;
}

// x joined over the lanes that are equal modulo W (W a power of two): rotations within 16 lanes, then swaps.
template <int W, class OP>
__device__ __forceinline__ float stride_join(float x) {
  if constexpr (W <= 8) x = OP::of(x, dpp_f32<0x128>(x));  // row_ror:8
  if constexpr (W <= 4) x = OP::of(x, dpp_f32<0x124>(x));
  if constexpr (W <= 2) x = OP::of(x, dpp_f32<0x122>(x));
  if constexpr (W <= 1) x = OP::of(x, dpp_f32<0x121>(x));
  if constexpr (W <= 16) x = join16<OP>(x);
  if constexpr (W <= 32) x = join32<OP>(x);
  return x;
}

// Distance buckets: map[clamp(d, -radius, radius) + radius] (map staged with its entries within the table).
// The distance saturates, so positions of any int32 value are in order.
__device__ __forceinline__ int distance_bucket(const unsigned char* map, int radius, int kpos, int qpos) {
  const int d = __builtin_elementwise_sub_sat(kpos, qpos);
  return map[max(-radius, min(radius, d)) + radius];
}

// Adds to two of a lane's own sums in LDS, [bucket][64 lanes]: no two lanes share a word or a bank, and the
// order is that of the program. Reading, adding and writing takes 8 clk of a CU for a wave, ds_add_f32 193. The
// second read does not wait for the first write; where both are one word the sum is carried over.
template <class A>
__device__ __forceinline__ void add_pair(A* mine, int t0, A x0, int t1, A x1) {
  A* const p0 = mine + 64 * t0;
  A* const p1 = mine + 64 * t1;
  const A a = *p0, b = *p1;
  x0 += a;
  x1 += t1 == t0 ? x0 : b;
  *p0 = x0;
  *p1 = x1;
}

inline bool aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
inline int launched() { return hipGetLastError() == hipSuccess ? FX_OK : FX_ERR_LAUNCH; }
inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline size_t dtype_size(int32_t dtype) {
  switch (dtype) {
    case FX_F32: return 4;
    case FX_F64: return 8;
    case FX_BF16:
    case FX_F16: return 2;
    default: return 0;
  }
}

// f(T{}) with the element type of dtype; FX_ERR_UNSUPPORTED for another.
template <bool F64, class F>
inline int with_type(int32_t dtype, F&& f) {
  switch (dtype) {
    case FX_F32: return f(float{});
    case FX_BF16: return f(__bf16{});
    case FX_F16: return f(_Float16{});
    case FX_F64:
      if constexpr (F64) return f(double{});
      return FX_ERR_UNSUPPORTED;
    default: return FX_ERR_INVALID_ARGUMENT;
  }
}

}  // namespace net
}  // namespace fx
