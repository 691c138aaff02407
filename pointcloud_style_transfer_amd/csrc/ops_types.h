// Element types and 8-wide row accesses shared by the block operators (rms_norm.hip,
// gated_linear.hip, grad_clip.hip).
#pragma once
#include "common.h"

namespace pcst {

// element type codes at the C boundary (include/pcst.h: PCST_F32 ..)
enum : int { kF32 = PCST_F32, kBF16 = PCST_BF16, kF16 = PCST_F16, kE4M3 = PCST_E4M3 };

struct EF32 {
  typedef float T;
};
struct EBF16 {
  typedef __bf16 T;
};
struct EF16 {
  typedef _Float16 T;
};
struct EE4M3 {
  typedef uint8_t T;
};

template <class T>
__device__ __forceinline__ float to_f32(T v) {
  return (float)v;
}

// 8 (4) consecutive elements at any element-aligned address as vector accesses (the hardware takes
// global accesses of any alignment), the first n elementwise where the row ends inside.  Vector types,
// not arrays: an array's eight elements are split up again and leave as narrow accesses.
template <class T, int N>
struct Vec {
  typedef T V __attribute__((ext_vector_type(N)));
  typedef V Any __attribute__((aligned(sizeof(T))));
};

template <class T, int N>
__device__ __forceinline__ void load_n(const T* p, int n, float (&v)[N]) {
  if (n >= N) {
    const typename Vec<T, N>::V q = *reinterpret_cast<const typename Vec<T, N>::Any*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)q[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < n ? (float)p[i] : 0.0f;
  }
}

template <class T, int N>
__device__ __forceinline__ void store_n(T* p, int n, const float (&v)[N]) {
  if (n >= N) {
    typename Vec<T, N>::V q;
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = (T)v[i];
    *reinterpret_cast<typename Vec<T, N>::Any*>(p) = q;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = (T)v[i];
  }
}

template <class T>
__device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
  load_n<T, 8>(p, n, v);
}
template <class T>
__device__ __forceinline__ void store8(T* p, int n, const float (&v)[8]) {
  store_n<T, 8>(p, n, v);
}

// 8 floats -> 8 e4m3 values (round to nearest even); NaN stays NaN
__device__ __forceinline__ uint2 pack8_e4m3(const float (&v)[8]) {
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}

}  // namespace pcst
