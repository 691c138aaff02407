// Root-mean-square norm of a residual stream, forward and backward, and the 8-bit row quantiser.
//
//   s = round_T(x + r)            (r given; else s = x)         the stream as it is stored
//   rho = 1 / sqrt(mean_d s^2 + eps)
//   y = s * rho * w               -> T, or
//   sc = max_d |y| / 448 (1 where that is 0),  q = e4m3(y / sc)
//
// Backward, a = w * dy, n = s * rho:   dx = dr = rho * (a - n * mean_d(a * n)) + ds
//                                      dw = sum over rows of dy * n
//
// Every row is read once: TPR threads hold it in registers (8 * NV values each) between the row sums
// and the output.  Sums and statistics are fp32; s is rounded to T because it is stored in T, and the
// norm is that of the stored stream, so the backward, which reads s again, normalises the same values.
// Bound by HBM, whose copy rate is 5.2 TB/s (1 GiB): 120000 x 256 fp16 with a residual 41.6 us (5.9 TB/s, part of
// the reads from the last-level cache), 8191 x 4096 bf16 50.8 us, the 8-bit form of 4096 x 4096 24.3 us; backward 45.7
// and 48.3 us, and 4 to 6 us for dw's second launch.  A few rows are one launch of 4 us.  dw: each work-group keeps its rows' column sums in registers, writes them as one
// partial row, and a second launch adds the partial rows in a fixed order (no atomics: deterministic).
#include "ops_types.h"

namespace pcst {
namespace {

constexpr int kNormMaxD = 16384;
// partial rows of dw: enough work-groups to keep HBM busy, few enough that the partials stay small next to
// the operands (4 bytes a column each, written and read once)
constexpr int kNormParts = 512, kNormPartsNarrow = 2048, kNormNarrow = 512;

template <int TPR>
__device__ __forceinline__ float row_reduce(float v, bool maximum, float* red) {
  constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    const float t = __shfl_xor(v, o, 64);
    v = maximum ? fmaxf(v, t) : v + t;
  }
  if (TPR > 64) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();  // the previous use of `red` has been read
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < TPR / 64; ++i) v = maximum ? fmaxf(v, red[i]) : v + red[i];
  }
  return v;
}

// w as floats for the columns of this thread
template <int TPR, int NV>
__device__ __forceinline__ void load_w(const void* w, int w_f32, int wt, int D, int c0,
                                       float (&wv)[NV][8]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = c0 + i * TPR * 8;
    const int n = D - c;
    if (n <= 0 || w == nullptr) {
#pragma unroll
      for (int k = 0; k < 8; ++k) wv[i][k] = 1.0f;
    } else if (w_f32) {
      load8(static_cast<const float*>(w) + c, n, wv[i]);
    } else if (wt == kBF16) {
      load8(static_cast<const __bf16*>(w) + c, n, wv[i]);
    } else {
      load8(static_cast<const _Float16*>(w) + c, n, wv[i]);
    }
  }
}

struct NormArgs {
  const void *x, *r, *w;
  int w_f32, wt;
  int64_t M;
  int D;
  float eps;
  void *y, *s;
  float *scale, *rho;
};

// QUANT: 0 y in T, 1 e4m3 + scale; NORM false: quantise x itself (no norm, no weight)
template <class T, int TPR, int NV, int QUANT, bool NORM>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_fwd_kernel(NormArgs a) {
  constexpr int kThreads = TPR > 256 ? TPR : 256;
  constexpr int RPB = kThreads / TPR;
  __shared__ float red[8];
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int c0 = lane * 8, D = a.D;
  const T* x = static_cast<const T*>(a.x);
  const T* r = static_cast<const T*>(a.r);
  float wv[NV][8];
  if (NORM) load_w<TPR, NV>(a.w, a.w_f32, a.wt, D, c0, wv);
  // rows of one work-group leave together: every thread of a row runs the same number of rounds
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.M; row0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = row0 + sub;
    const bool live = row < a.M;
    const int64_t at = (live ? row : row0) * D;
    float v[NV][8];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = c0 + i * TPR * 8, n = D - c;
      if (n > 0) {
        load8(x + at + c, n, v[i]);
        if (r) {
          float t[8];
          load8(r + at + c, n, t);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[i][k] = (float)(T)(v[i][k] + t[k]);
          if (live) store8(static_cast<T*>(a.s) + at + c, n, v[i]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = 0.0f;
      }
      if (NORM) {
#pragma unroll
        for (int k = 0; k < 8; ++k) ss = fmaf(v[i][k], v[i][k], ss);
      }
    }
    if (NORM) {
      ss = row_reduce<TPR>(ss, false, red);
      const float rho = 1.0f / sqrtf(ss / (float)D + a.eps);
      if (a.rho && live && lane == 0) a.rho[row] = rho;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = v[i][k] * rho * wv[i][k];
    }
    if (QUANT) {
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) top = c0 + i * TPR * 8 + k < D ? fmaxf(top, fabsf(v[i][k])) : top;
      top = row_reduce<TPR>(top, true, red);
      const float sc = top > 0.0f ? top / 448.0f : 1.0f;
      const float inv = 1.0f / sc;
      const bool plain = !(sc > 0x1p-100f && sc < 0x1p100f);
      if (live && lane == 0) a.scale[row] = sc;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * TPR * 8, n = D - c;
        if (n <= 0 || !live) continue;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          // the quotient from the reciprocal and one correction; the division itself for scales whose
          // reciprocal is no normal number
          const float q0 = v[i][k] * inv;
          v[i][k] = plain ? v[i][k] / sc : fmaf(fmaf(-q0, sc, v[i][k]), inv, q0);
        }
        const uint2 q = pack8_e4m3(v[i]);
        uint8_t* out = static_cast<uint8_t*>(a.y) + at + c;
        if (n >= 8) {
          struct __attribute__((packed, aligned(1))) P { uint32_t x, y; };
          *reinterpret_cast<P*>(out) = P{q.x, q.y};
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < n) out[k] = (uint8_t)((k < 4 ? q.x : q.y) >> (8 * (k & 3)));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * TPR * 8, n = D - c;
        if (n > 0 && live) store8(static_cast<T*>(a.y) + at + c, n, v[i]);
      }
    }
  }
}

struct NormBwdArgs {
  const void *s, *w, *dy, *ds;
  const float* rho;
  int w_f32, wt;
  int64_t M;
  int D;
  void* dx;
  float* part;  // [gridDim.x, D] or null
};

// 8 values as they are stored, the first n of them, zeros behind
template <class T>
__device__ __forceinline__ typename Vec<T, 8>::V raw8(const T* p, int n) {
  if (n >= 8) return *reinterpret_cast<const typename Vec<T, 8>::Any*>(p);
  typename Vec<T, 8>::V v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : (T)0.0f;
  return v;
}

// One row of s, dy and ds in flight while the previous one is worked on: with few work-groups (each
// leaves a partial row of dw) the loads of one row at a time keep too little of HBM busy.
template <class T, int TPR, int NV>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_bwd_kernel(NormBwdArgs a) {
  typedef typename Vec<T, 8>::V V;
  constexpr int kThreads = TPR > 256 ? TPR : 256;
  constexpr int RPB = kThreads / TPR;
  constexpr bool AHEAD = NV < 4;  // (the widest rows have no registers left for it)
  __shared__ float red[8];
  __shared__ float cs[RPB > 1 ? TPR * NV * 8 : 1];
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int c0 = lane * 8, D = a.D;
  const T* sp = static_cast<const T*>(a.s);
  const T* dyp = static_cast<const T*>(a.dy);
  const T* dsp = static_cast<const T*>(a.ds);
  float wv[NV][8], acc[NV][8];
  load_w<TPR, NV>(a.w, a.w_f32, a.wt, D, c0, wv);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[i][k] = 0.0f;
  V sv[NV], gv[NV], dv[NV];
  float rho = 0.0f;
  auto fetch = [&](int64_t row, bool live) {
    rho = live ? a.rho[row] : 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = c0 + i * TPR * 8, n = live ? D - c : 0;
      const int64_t at = row * D + c;
      sv[i] = n > 0 ? raw8(sp + at, n) : V{};
      gv[i] = n > 0 ? raw8(dyp + at, n) : V{};
      dv[i] = n > 0 && dsp ? raw8(dsp + at, n) : V{};
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + sub;
  if (AHEAD) fetch(row, row < a.M);
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.M; row0 += step, row += step) {
    const bool live = row < a.M;
    if (!AHEAD) fetch(row, live);
    float n_[NV][8], g[NV][8], o[NV][8];
    float dot = 0.0f;
    const float r = rho;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        n_[i][k] = (float)sv[i][k] * r;
        g[i][k] = (float)gv[i][k];
        o[i][k] = (float)dv[i][k];
      }
    if (AHEAD && row0 + step < a.M) fetch(row + step, row + step < a.M);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) {  // (a row past the end is all zeros)
        acc[i][k] = fmaf(g[i][k], n_[i][k], acc[i][k]);
        g[i][k] *= wv[i][k];
        dot = fmaf(g[i][k], n_[i][k], dot);
      }
    if (!a.dx) continue;
    const float c1 = row_reduce<TPR>(dot, false, red) / (float)D;
    if (!live) continue;  // (no barrier is skipped: more than one row a work-group means none is used)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = c0 + i * TPR * 8, n = D - c;
      if (n <= 0) continue;
#pragma unroll
      for (int k = 0; k < 8; ++k) o[i][k] += r * (g[i][k] - n_[i][k] * c1);
      store8(static_cast<T*>(a.dx) + row * D + c, n, o[i]);
    }
  }
  if (!a.part) return;
  float* part = a.part + (int64_t)blockIdx.x * D;
  if (RPB > 1) {  // the rows of the work-group meet in LDS, in order
    for (int q = 0; q < RPB; ++q) {
      if (sub == q) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float* p = &cs[(i * TPR + lane) * 8 + k];
            *p = q ? *p + acc[i][k] : acc[i][k];
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < D; c += kThreads) part[c] = cs[c];
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = c0 + i * TPR * 8, n = D - c;
      if (n > 0) store8(part + c, n, acc[i]);
    }
  }
}

// dw[d] = sum over the partial rows, 16 columns a work-group, 64 slices of the rows, fp64, in a fixed order
__global__ __launch_bounds__(1024) void norm_dw_kernel(const float* __restrict__ part, int parts, int D,
                                                       void* dw, int dwt) {
  __shared__ double red[64][17];
  const int c = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int d = blockIdx.x * 16 + c;
  double s = 0.0;
  if (d < D) {
#pragma unroll 8
    for (int p = q; p < parts; p += 64) s += (double)part[(int64_t)p * D + d];
  }
  red[q][c] = s;
  __syncthreads();
  if (q < 8) {
    for (int i = q + 8; i < 64; i += 8) s += red[i][c];
  }
  __syncthreads();
  if (q < 8) red[q][c] = s;
  __syncthreads();
  if (q == 0 && d < D) {
    for (int i = 1; i < 8; ++i) s += red[i][c];
    if (dwt == kF32)
      static_cast<float*>(dw)[d] = (float)s;
    else if (dwt == kBF16)
      static_cast<__bf16*>(dw)[d] = (__bf16)(float)s;
    else
      static_cast<_Float16*>(dw)[d] = (_Float16)(float)s;
  }
}

// threads per row and 8-value groups per thread: a row within one wave up to 1024 columns (its sums
// need no barrier), a work-group beyond
#define PCST_NORM_SHAPES(D, CALL)      \
  do {                                 \
    if ((D) <= 128) CALL(16, 1);       \
    else if ((D) <= 256) CALL(32, 1);  \
    else if ((D) <= 512) CALL(64, 1);  \
    else if ((D) <= 1024) CALL(64, 2); \
    else if ((D) <= 2048) CALL(256, 1); \
    else if ((D) <= 4096) CALL(256, 2); \
    else if ((D) <= 8192) CALL(512, 2); \
    else CALL(512, 4);                 \
  } while (0)

int norm_rpb(int64_t D) { return D <= 128 ? 16 : D <= 256 ? 8 : D <= 1024 ? 4 : 1; }

template <class T, int QUANT, bool NORM>
void launch_fwd(const NormArgs& a, hipStream_t s) {
  const unsigned grid = (unsigned)std::min<int64_t>(cdiv(a.M, norm_rpb(a.D)), 4096);
#define CALL(TPR, NV)                                                                          \
  hipLaunchKernelGGL((norm_fwd_kernel<T, TPR, NV, QUANT, NORM>), dim3(grid),                   \
                     dim3(TPR > 256 ? TPR : 256), 0, s, a)
  PCST_NORM_SHAPES(a.D, CALL);
#undef CALL
}

template <class T>
void launch_bwd(const NormBwdArgs& a, unsigned grid, hipStream_t s) {
#define CALL(TPR, NV) \
  hipLaunchKernelGGL((norm_bwd_kernel<T, TPR, NV>), dim3(grid), dim3(TPR > 256 ? TPR : 256), 0, s, a)
  PCST_NORM_SHAPES(a.D, CALL);
#undef CALL
}

bool is_float(int t) { return t == kF32 || t == kBF16 || t == kF16; }

int64_t norm_parts(int64_t M, int64_t D) {
  return std::min<int64_t>(cdiv(M, norm_rpb(D)), D <= kNormNarrow ? kNormPartsNarrow : kNormParts);
}

int check_dims(const char* who, int64_t M, int64_t D, int dt, int wdt) {
  PCST_CHECK_ARG(M >= 0 && D > 0, "%s: bad shape M=%lld D=%lld", who, (long long)M, (long long)D);
  PCST_CHECK_ARG(is_float(dt) && (wdt == dt || wdt == kF32),
                 "%s: x is float32, bfloat16 or float16 and the weight of its type or float32", who);
  if (D > kNormMaxD) {
    set_error("%s: rows of %lld values, at most %d", who, (long long)D, kNormMaxD);
    return PCST_EUNSUPPORTED;
  }
  return PCST_OK;
}

}  // namespace
}  // namespace pcst

using namespace pcst;

extern "C" int pcst_rms_norm(const void* x, const void* residual, int dtype, int64_t M, int64_t D,
                             const void* weight, int weight_dtype, float eps, void* y, void* s,
                             float* rho, void* stream) {
  if (int rc = check_dims("rms_norm", M, D, dtype, weight_dtype)) return rc;
  if (M == 0) return PCST_OK;
  PCST_CHECK_ARG(x && weight && y && (!residual || s), "rms_norm: null pointer");
  const NormArgs a{x, residual, weight, weight_dtype == kF32, dtype, M, (int)D, eps, y, s, nullptr, rho};
  hipStream_t st = as_stream(stream);
  if (dtype == kF32) launch_fwd<float, 0, true>(a, st);
  else if (dtype == kBF16) launch_fwd<__bf16, 0, true>(a, st);
  else launch_fwd<_Float16, 0, true>(a, st);
  PCST_LAUNCH_CHECK("rms_norm");
  return PCST_OK;
}

extern "C" int pcst_rms_norm_quant(const void* x, const void* residual, int dtype, int64_t M,
                                   int64_t D, const void* weight, int weight_dtype, float eps,
                                   void* q, float* scale, void* s, void* stream) {
  if (int rc = check_dims("rms_norm_quant", M, D, dtype, weight_dtype)) return rc;
  if (M == 0) return PCST_OK;
  PCST_CHECK_ARG(x && weight && q && scale && (!residual || s), "rms_norm_quant: null pointer");
  const NormArgs a{x, residual, weight, weight_dtype == kF32, dtype, M, (int)D, eps, q, s, scale, nullptr};
  hipStream_t st = as_stream(stream);
  if (dtype == kF32) launch_fwd<float, 1, true>(a, st);
  else if (dtype == kBF16) launch_fwd<__bf16, 1, true>(a, st);
  else launch_fwd<_Float16, 1, true>(a, st);
  PCST_LAUNCH_CHECK("rms_norm_quant");
  return PCST_OK;
}

extern "C" int pcst_quant_rows(const void* x, int dtype, int64_t M, int64_t D, void* q, float* scale,
                               void* stream) {
  if (int rc = check_dims("quant_rows", M, D, dtype, kF32)) return rc;
  if (M == 0) return PCST_OK;
  PCST_CHECK_ARG(x && q && scale, "quant_rows: null pointer");
  const NormArgs a{x, nullptr, nullptr, 1, dtype, M, (int)D, 0.0f, q, nullptr, scale, nullptr};
  hipStream_t st = as_stream(stream);
  if (dtype == kF32) launch_fwd<float, 1, false>(a, st);
  else if (dtype == kBF16) launch_fwd<__bf16, 1, false>(a, st);
  else launch_fwd<_Float16, 1, false>(a, st);
  PCST_LAUNCH_CHECK("quant_rows");
  return PCST_OK;
}

extern "C" int pcst_rms_norm_bwd_workspace_size(int64_t M, int64_t D, size_t* bytes) {
  PCST_CHECK_ARG(M >= 0 && D > 0 && bytes, "rms_norm_bwd_workspace_size: bad args");
  *bytes = sizeof(float) * (size_t)norm_parts(M, D) * (size_t)D;
  return PCST_OK;
}

extern "C" int pcst_rms_norm_bwd(const void* s, int dtype, int64_t M, int64_t D, const void* weight,
                                 int weight_dtype, const float* rho, const void* dy, const void* ds,
                                 void* dx, void* dw, void* workspace, void* stream) {
  if (int rc = check_dims("rms_norm_bwd", M, D, dtype, weight_dtype)) return rc;
  PCST_CHECK_ARG(weight && (M == 0 || (s && rho && dy)) && (!dw || M == 0 || workspace),
                 "rms_norm_bwd: null pointer");
  hipStream_t st = as_stream(stream);
  const int64_t parts = norm_parts(M, D);
  if (M > 0 && (dx || dw)) {
    const NormBwdArgs a{s, weight, dy, ds, rho, weight_dtype == kF32, dtype, M, (int)D, dx,
                        dw ? static_cast<float*>(workspace) : nullptr};
    if (dtype == kF32) launch_bwd<float>(a, (unsigned)parts, st);
    else if (dtype == kBF16) launch_bwd<__bf16>(a, (unsigned)parts, st);
    else launch_bwd<_Float16>(a, (unsigned)parts, st);
  }
  if (dw)
    hipLaunchKernelGGL(norm_dw_kernel, dim3((unsigned)cdiv(D, 16)), dim3(1024), 0, st,
                       static_cast<const float*>(workspace), (int)parts, (int)D, dw, weight_dtype);
  PCST_LAUNCH_CHECK("rms_norm_bwd");
  return PCST_OK;
}
