// The global norm of many gradient tensors, and clipping by it.
//
//   N = inv * (sum over all tensors of |g|^p)^(1/p),  p = 1, 2 or inf
//   c = min(1, max_norm / (N + 1e-6)) * inv,          out = g * c
//
// Two launches (per 128 tensors): the norm's, whose work-groups each leave one partial in fp64, and
// the scaling's, whose work-groups each add all partials in the same fixed order themselves -- at most
// 1024 a launch, so that no third launch, no atomic and no zeroed counter stands between.  fp64 sums: a
// square of any finite float is finite there, and their order does not show in the 24 bits returned.  The
// tensors' addresses travel in the kernel arguments, so a captured launch keeps them.  Bound by HBM: every gradient is read twice and written once (268M fp16: 356 us, 4.5 TB/s); a
// model's 80 tensors of 2.5M values are two launches of 8 us.
#include <algorithm>
#include <type_traits>
#include <utility>
#include <vector>

#include "ops_types.h"

namespace pcst {
namespace {

constexpr int kClipTensors = 128;  // per launch: 128 * 29 bytes of kernel arguments

struct ClipTable {
  const void* in[kClipTensors];
  void* out[kClipTensors];
  int64_t n[kClipTensors];
  int32_t first[kClipTensors + 1];  // a tensor's first chunk
  uint8_t type[kClipTensors];       // element type code, the output's in the high half
  int32_t count;
};

// chunk of this work-group -> (tensor, element range)
__device__ __forceinline__ int find_tensor(const ClipTable& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// the larger one, NaN where either is one
__device__ __forceinline__ double nan_max(double a, double b) { return (b > a || b != b) ? b : a; }

__device__ __forceinline__ double wave_total(double v, int p) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const double t = __shfl_xor(v, o, 64);
    v = p == 0 ? nan_max(v, t) : v + t;
  }
  return v;
}

// all 256 threads' values together, in the same order on every thread
__device__ __forceinline__ double block_total(double v, int p, double* red) {
  v = wave_total(v, p);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = red[0];
#pragma unroll
  for (int i = 1; i < 4; ++i) s = p == 0 ? nan_max(s, red[i]) : s + red[i];
  return s;
}

__device__ __forceinline__ double add_term(double s, float v, int p) {
  const double d = (double)v;
  return p == 2 ? fma(d, d, s) : p == 1 ? s + fabs(d) : nan_max(s, fabs(d));
}

// 8 values.  A 16-bit value's square is exact in fp32: four of them are added there, two roundings of 2^-24 of
// their sum, and fp64 adds the fours (268M fp16, whose norm waits for fp64's instructions: 382 -> 357 us).
// bf16 squares may leave fp32's range on either side; such fours go the way of fp32's values.
template <class V>
__device__ __forceinline__ double add_piece(double s, V v, int p) {
  constexpr bool kF = std::is_same<V, Vec<_Float16, 8>::V>::value, kB = std::is_same<V, Vec<__bf16, 8>::V>::value;
#pragma unroll
  for (int j = 0; j < 8; j += 4) {
    const float a = (float)v[j], b = (float)v[j + 1], c = (float)v[j + 2], d = (float)v[j + 3];
    const float q = fmaf(b, b, a * a) + fmaf(d, d, c * c);
    if ((kF || kB) && p == 2 && (kF || (q > 0x1p-100f && q < 0x1p120f))) {
      s += (double)q;
    } else {
      s = add_term(add_term(add_term(add_term(s, a, p), b, p), c, p), d, p);
    }
  }
  return s;
}

constexpr int kFlight = 4;  // 8-value pieces a thread has in flight

template <class T>
__device__ __forceinline__ double range_sum(const T* g, int64_t lo, int64_t hi, int p, double s) {
  typedef typename Vec<T, 8>::V V;
  int64_t i = lo + threadIdx.x * 8;
  for (; i + (kFlight - 1) * 2048 + 8 <= hi; i += kFlight * 2048) {
    V v[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) v[u] = *reinterpret_cast<const typename Vec<T, 8>::Any*>(g + i + u * 2048);
#pragma unroll
    for (int u = 0; u < kFlight; ++u) s = add_piece(s, v[u], p);
  }
  for (; i < hi; i += 2048) {
    float v[8];
    load8(g + i, (int)(hi - i < 8 ? hi - i : 8), v);  // zeros past the end add nothing
#pragma unroll
    for (int j = 0; j < 8; ++j) s = add_term(s, v[j], p);
  }
  return s;
}

__global__ __launch_bounds__(256) void grad_norm_kernel(ClipTable t, int64_t chunk_len, int p,
                                                        double* __restrict__ part) {
  __shared__ double red[4];
  double s = 0.0;
  for (int c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
    const int k = find_tensor(t, c);
    const int64_t lo = (int64_t)(c - t.first[k]) * chunk_len;
    const int64_t hi = lo + chunk_len < t.n[k] ? lo + chunk_len : t.n[k];
    const int type = t.type[k] & 15;
    if (type == kF32) s = range_sum(static_cast<const float*>(t.in[k]), lo, hi, p, s);
    else if (type == kBF16) s = range_sum(static_cast<const __bf16*>(t.in[k]), lo, hi, p, s);
    else s = range_sum(static_cast<const _Float16*>(t.in[k]), lo, hi, p, s);
  }
  s = block_total(s, p, red);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

template <class T, class O>
__device__ __forceinline__ void range_scale(const T* g, O* o, int64_t lo, int64_t hi, float f) {
  typedef typename Vec<T, 8>::V V;
  int64_t i = lo + threadIdx.x * 8;
  for (; i + (kFlight - 1) * 2048 + 8 <= hi; i += kFlight * 2048) {
    V v[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) v[u] = *reinterpret_cast<const typename Vec<T, 8>::Any*>(g + i + u * 2048);
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = (float)v[u][j] * f;
      store8(o + i + u * 2048, 8, w);
    }
  }
  for (; i < hi; i += 2048) {
    const int n = (int)(hi - i < 8 ? hi - i : 8);
    float v[8];
    load8(g + i, n, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= f;
    store8(o + i, n, v);
  }
}

__global__ __launch_bounds__(256) void grad_scale_kernel(ClipTable t, int64_t chunk_len, int p,
                                                         const double* __restrict__ part, int parts,
                                                         double max_norm, const float* inv_scale,
                                                         float* __restrict__ norm) {
  __shared__ double red[4];
  double s = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < parts; i += 256) s = p == 0 ? nan_max(s, part[i]) : s + part[i];
  s = block_total(s, p, red);
  const double inv = inv_scale ? (double)*inv_scale : 1.0;
  const double total = (p == 2 ? sqrt(s) : s) * fabs(inv);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
  double q = max_norm / (total + 1e-6);
  q = q > 1.0 ? 1.0 : q;  // NaN stays
  const float f = (float)(q * inv);
  // from the last chunk down: what the norm's launch read last is still in the caches
  for (int b = blockIdx.x; b < t.first[t.count]; b += gridDim.x) {
    const int c = t.first[t.count] - 1 - b;
    const int k = find_tensor(t, c);
    if (f == 1.0f && t.in[k] == t.out[k]) continue;  // g * 1 is g
    const int64_t lo = (int64_t)(c - t.first[k]) * chunk_len;
    const int64_t hi = lo + chunk_len < t.n[k] ? lo + chunk_len : t.n[k];
    const void* g = t.in[k];
    void* o = t.out[k];
    switch (t.type[k]) {
      case kF32 | kF32 << 4: range_scale(static_cast<const float*>(g), static_cast<float*>(o), lo, hi, f); break;
      case kBF16 | kBF16 << 4: range_scale(static_cast<const __bf16*>(g), static_cast<__bf16*>(o), lo, hi, f); break;
      case kF16 | kF16 << 4: range_scale(static_cast<const _Float16*>(g), static_cast<_Float16*>(o), lo, hi, f); break;
      case kBF16 | kF32 << 4: range_scale(static_cast<const __bf16*>(g), static_cast<float*>(o), lo, hi, f); break;
      default: range_scale(static_cast<const _Float16*>(g), static_cast<float*>(o), lo, hi, f); break;
    }
  }
}

// A chunk is what a work-group takes at a time; a launch has at most kClipGroups work-groups (4 a CU, each
// thread with kFlight loads in flight), which take chunk after chunk and leave one partial each.
constexpr int kClipGroups = 1024;
int64_t clip_chunk(int64_t total) {
  return std::max<int64_t>(2048, std::min<int64_t>(16384, cdiv(cdiv(total, kClipGroups), 2048) * 2048));
}

int64_t clip_total(const int64_t* n, int count) {
  int64_t t = 0;
  for (int i = 0; i < count; ++i) t += n[i];
  return t;
}

// partials of all launches
int64_t clip_parts(const int64_t* n, int count, int64_t chunk) {
  int64_t parts = 0, c = 0;
  int in = 0;
  for (int i = 0; i < count; ++i) {
    if (n[i] == 0) continue;
    c += cdiv(n[i], chunk);
    if (++in == kClipTensors) {
      parts += std::min<int64_t>(c, kClipGroups);
      in = 0;
      c = 0;
    }
  }
  return parts + std::min<int64_t>(c, kClipGroups);
}

template <class F>
void for_tables(const void* const* in, void* const* out, const int64_t* n, const uint8_t* type, int count,
                int64_t chunk, F f) {
  int64_t base = 0;
  for (int i = 0; i < count;) {
    ClipTable t;
    t.count = 0;
    int32_t c = 0;
    for (; i < count && t.count < kClipTensors; ++i) {
      if (n[i] == 0) continue;
      t.in[t.count] = in[i];
      t.out[t.count] = out ? out[i] : nullptr;
      t.n[t.count] = n[i];
      t.type[t.count] = type[i];
      t.first[t.count++] = c;
      c += (int32_t)cdiv(n[i], chunk);
    }
    if (t.count == 0) break;
    t.first[t.count] = c;
    const int32_t groups = std::min<int32_t>(c, kClipGroups);
    f(t, groups, base);
    base += groups;
  }
}

// the norm alone (no outputs)
__global__ __launch_bounds__(256) void grad_total_kernel(const double* __restrict__ part, int parts, int p,
                                                         const float* inv_scale, float* __restrict__ norm) {
  __shared__ double red[4];
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) s = p == 0 ? nan_max(s, part[i]) : s + part[i];
  s = block_total(s, p, red);
  if (threadIdx.x == 0) *norm = (float)((p == 2 ? sqrt(s) : s) * fabs(inv_scale ? (double)*inv_scale : 1.0));
}

// whether two of the tensors' byte ranges overlap (a gradient written in place counts once)
bool overlap(const void* const* in, void* const* out, const int64_t* n, const uint8_t* type, int count) {
  std::vector<std::pair<uintptr_t, uintptr_t>> r;
  r.reserve(2 * (size_t)count);
  auto add = [&](const void* p, int64_t len, int t) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    r.emplace_back(a, a + (uintptr_t)len * (t == kF32 ? 4 : 2));
  };
  for (int i = 0; i < count; ++i) {
    if (n[i] == 0) continue;
    add(in[i], n[i], type[i] & 15);
    if (out && (out[i] != in[i] || (type[i] & 15) != type[i] >> 4)) add(out[i], n[i], type[i] >> 4);
  }
  std::sort(r.begin(), r.end());
  for (size_t i = 1; i < r.size(); ++i)
    if (r[i].first < r[i - 1].second) return true;
  return false;
}

bool is_float(int t) { return t == kF32 || t == kBF16 || t == kF16; }

}  // namespace
}  // namespace pcst

using namespace pcst;

extern "C" int pcst_grad_clip_workspace_size(const int64_t* numel, int count, size_t* bytes) {
  PCST_CHECK_ARG(count >= 0 && (count == 0 || numel) && bytes, "grad_clip_workspace_size: bad args");
  *bytes = sizeof(double) * (size_t)std::max<int64_t>(1, clip_parts(numel, count, clip_chunk(clip_total(numel, count))));
  return PCST_OK;
}

extern "C" int pcst_grad_clip(const void* const* grads, void* const* out, const int64_t* numel,
                              const uint8_t* types, int count, int norm_p, double max_norm,
                              const float* inv_scale, float* norm, void* workspace, void* stream) {
  PCST_CHECK_ARG(count >= 0 && (count == 0 || (grads && numel && types)) && norm, "grad_clip: null pointer");
  PCST_CHECK_ARG(norm_p >= 0 && norm_p <= 2, "grad_clip: norm_p is 1, 2 or 0 (the largest absolute value)");
  PCST_CHECK_ARG(max_norm >= 0, "grad_clip: max_norm is at least 0");
  for (int i = 0; i < count; ++i) {
    const int ti = types[i] & 15, to = types[i] >> 4;
    PCST_CHECK_ARG(is_float(ti) && (to == ti || to == kF32),
                   "grad_clip: tensor %d: gradients are float32, bfloat16 or float16, outputs of their type or float32", i);
    PCST_CHECK_ARG(numel[i] >= 0 && (numel[i] == 0 || (grads[i] && (!out || out[i]))),
                   "grad_clip: tensor %d: bad size or null pointer", i);
  }
  const int64_t total = clip_total(numel, count);
  PCST_CHECK_ARG(total < (1ll << 40), "grad_clip: too many elements");
  bool clash = false;
  try {
    clash = overlap(grads, out, numel, types, count);
  } catch (...) {  // nothing is thrown across the C boundary
    set_error("grad_clip: no host memory for %d tensors", count);
    return PCST_EINVAL;
  }
  PCST_CHECK_ARG(!clash, "grad_clip: two of the tensors overlap (or one is given twice)");
  hipStream_t s = as_stream(stream);
  PCST_CHECK_ARG(total == 0 || workspace, "grad_clip: null workspace");
  double* part = static_cast<double*>(workspace);
  const int64_t chunk = clip_chunk(total);
  const int parts = (int)clip_parts(numel, count, chunk);
  for_tables(grads, out, numel, types, count, chunk, [&](const ClipTable& t, int32_t c, int64_t base) {
    hipLaunchKernelGGL(grad_norm_kernel, dim3((unsigned)c), dim3(256), 0, s, t, chunk, norm_p, part + base);
  });
  if (!out || parts == 0) {
    hipLaunchKernelGGL(grad_total_kernel, dim3(1), dim3(256), 0, s, part, parts, norm_p, inv_scale, norm);
    PCST_LAUNCH_CHECK("grad_clip");
    return PCST_OK;
  }
  for_tables(grads, out, numel, types, count, chunk, [&](const ClipTable& t, int32_t c, int64_t base) {
    hipLaunchKernelGGL(grad_scale_kernel, dim3((unsigned)c), dim3(256), 0, s, t, chunk, norm_p, part, parts,
                       max_norm, inv_scale, base ? nullptr : norm);
  });
  PCST_LAUNCH_CHECK("grad_clip");
  return PCST_OK;
}
