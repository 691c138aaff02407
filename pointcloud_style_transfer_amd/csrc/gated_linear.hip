// Gated linear layer, C entry points: checks, the layout of the workspace, and copies of operands whose
// rows are not whole 16-byte pieces.  The products are in gated_core.h.
#include "gated_core.h"

namespace pcst {
namespace {

int elem(int dt) { return dt == kF32 ? 4 : dt == kE4M3 ? 1 : 2; }

// rows of `cols` bytes -> rows of `pitch` bytes, the rest zero; 4 bytes (or less, at the end) a thread
__global__ void pad_rows_kernel(const uint8_t* __restrict__ src, int64_t rows, int64_t cols, int64_t pitch,
                                uint32_t* __restrict__ dst) {
  struct __attribute__((packed, aligned(1))) U { uint32_t v; };
  const int64_t pw = pitch / 4, n = rows * pw;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / pw, c = (i - r * pw) * 4;
    uint32_t v = 0;
    if (c + 4 <= cols) {
      v = reinterpret_cast<const U*>(src + r * cols + c)->v;
    } else {
      for (int k = 0; k < 4; ++k)
        if (c + k < cols) v |= (uint32_t)src[r * cols + c + k] << (8 * k);
    }
    dst[i] = v;
  }
}

void pad_rows(const void* src, int64_t rows, int64_t cols, int64_t pitch, void* dst, hipStream_t s) {
  const int64_t n = rows * (pitch / 4);
  hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)std::min<int64_t>(cdiv(n, 256), 4096)), dim3(256), 0, s,
                     static_cast<const uint8_t*>(src), rows, cols, pitch, static_cast<uint32_t*>(dst));
}

struct Layout {
  int64_t pitch;  // bytes of a padded row of D values
  void *x, *wg, *wu;
  void* dgu;
  float *bpart, *part;
  int64_t fpad;
  size_t bytes;
};

// pad: x, Wg and Wu (or some of them) need copies
Layout lay(void* ws, int dt, int64_t M, int64_t D, int64_t F, bool pad, bool bwd) {
  Layout l{};
  Carver c(ws);
  const int es = elem(dt);
  l.pitch = cdiv(D * es, 16) * 16;
  if (pad) {
    l.x = c.take<char>((size_t)(M * l.pitch));
    l.wg = c.take<char>((size_t)(F * l.pitch));
    l.wu = c.take<char>((size_t)(F * l.pitch));
  }
  l.fpad = cdiv(F, 64) * 64;
  if (bwd) {
    l.dgu = c.take<char>((size_t)(M * 2 * l.fpad * es));
    l.bpart = c.take<float>((size_t)(gated::bias_parts(M, D, F, es, gated::plan_gated(M, D, F, es)) * 2 * F));
  }
  l.part = c.take<float>((size_t)gated::part_floats(M, D, F, es, bwd));
  l.bytes = c.bytes();
  return l;
}

// operands as the products take them: rows of whole 16-byte pieces on 16-byte boundaries
bool ready(const void* p, int64_t D, int es) { return (D * es) % 16 == 0 && (uintptr_t)p % 16 == 0; }

int check(const char* who, int dt, int64_t M, int64_t D, int64_t F, int act) {
  PCST_CHECK_ARG(M >= 0 && D > 0 && F > 0, "%s: bad shape M=%lld D=%lld F=%lld", who, (long long)M, (long long)D, (long long)F);
  PCST_CHECK_ARG(dt >= kF32 && dt <= kE4M3, "%s: unknown element type %d", who, dt);
  PCST_CHECK_ARG(act >= 0 && act <= 2, "%s: act is 0 (silu), 1 (gelu) or 2 (relu)", who);
  // a tile's rows are addressed with 31 bits
  if (D >= (1 << 20) || F >= (1 << 20) || M >= (1ll << 31)) {
    set_error("%s: at most 2^20 - 1 features and 2^31 - 1 rows", who);
    return PCST_EUNSUPPORTED;
  }
  return PCST_OK;
}

// x, Wg, Wu into the call, padded copies where needed (one pitch for both weights)
void operands(gated::FwdCall& c, const Layout& l, const void* x, const void* wg, const void* wu, int es, hipStream_t s) {
  c.x = x;
  c.wg = wg;
  c.wu = wu;
  c.ldx = c.ldw = c.D * es;
  if (!ready(x, c.D, es)) {
    pad_rows(x, c.M, c.D * es, l.pitch, l.x, s);
    c.x = l.x;
    c.ldx = l.pitch;
  }
  if (!ready(wg, c.D, es) || !ready(wu, c.D, es)) {
    pad_rows(wg, c.F, c.D * es, l.pitch, l.wg, s);
    pad_rows(wu, c.F, c.D * es, l.pitch, l.wu, s);
    c.wg = l.wg;
    c.wu = l.wu;
    c.ldw = l.pitch;
  }
}

}  // namespace
}  // namespace pcst

using namespace pcst;

extern "C" int pcst_gated_linear_workspace_size(int dtype, int64_t M, int64_t D, int64_t F, int aligned,
                                                size_t* bytes) {
  if (int rc = check("gated_linear_workspace_size", dtype, M, D, F, 0)) return rc;
  PCST_CHECK_ARG(bytes, "gated_linear_workspace_size: null pointer");
  const bool pad = !aligned || (D * elem(dtype)) % 16 != 0;
  *bytes = gated::take_rows(M, D, F, elem(dtype)) ? 0 : lay(nullptr, dtype, M, D, F, pad, false).bytes;
  return PCST_OK;
}

extern "C" int pcst_gated_linear(const void* x, int dtype, int64_t M, int64_t D, const void* w_gate,
                                 const void* w_up, int64_t F, const void* b_gate, const void* b_up,
                                 int bias_f32, int act, const float* x_scale, const float* gate_scale,
                                 const float* up_scale, void* h, int out_dtype, void* workspace,
                                 void* stream) {
  if (int rc = check("gated_linear", dtype, M, D, F, act)) return rc;
  PCST_CHECK_ARG((b_gate == nullptr) == (b_up == nullptr), "gated_linear: both biases or none");
  if (dtype == kE4M3) {
    PCST_CHECK_ARG(out_dtype == kBF16 || out_dtype == kF16, "gated_linear: e4m3 operands give bfloat16 or float16");
    PCST_CHECK_ARG(M == 0 || (x_scale && gate_scale && up_scale), "gated_linear: e4m3 operands need their scales");
  } else {
    PCST_CHECK_ARG(out_dtype == dtype, "gated_linear: the output is of the operands' type");
  }
  if (M == 0) return PCST_OK;
  PCST_CHECK_ARG(x && w_gate && w_up && h, "gated_linear: null pointer");
  const int es = elem(dtype);
  const bool rows = gated::take_rows(M, D, F, es);
  const bool pad = !ready(x, D, es) || !ready(w_gate, D, es) || !ready(w_up, D, es);
  const Layout l = lay(workspace, dtype, M, D, F, pad, false);
  PCST_CHECK_ARG(rows || l.bytes == 0 || workspace, "gated_linear: null workspace");
  gated::FwdCall c{};
  c.M = M;
  c.D = D;
  c.F = F;
  if (rows) {
    c.x = x;
    c.wg = w_gate;
    c.wu = w_up;
    c.ldx = c.ldw = D * es;
  } else {
    operands(c, l, x, w_gate, w_up, es, as_stream(stream));
    c.part = l.part;
  }
  c.bg = b_gate;
  c.bu = b_up;
  c.bias_f32 = bias_f32;
  c.act = act;
  c.out_type = out_dtype;
  c.xs = x_scale;
  c.gs = gate_scale;
  c.us = up_scale;
  c.h = h;
  switch (dtype) {
    case kF32: return gated::fwd<EF32>(c, stream);
    case kBF16: return gated::fwd<EBF16>(c, stream);
    case kF16: return gated::fwd<EF16>(c, stream);
    default: return gated::fwd<EE4M3>(c, stream);
  }
}

extern "C" int pcst_gated_linear_bwd_workspace_size(int dtype, int64_t M, int64_t D, int64_t F, size_t* bytes) {
  if (int rc = check("gated_linear_bwd_workspace_size", dtype, M, D, F, 0)) return rc;
  PCST_CHECK_ARG(bytes && dtype != kE4M3, "gated_linear_bwd_workspace_size: bad args");
  *bytes = lay(nullptr, dtype, M, D, F, true, true).bytes;
  return PCST_OK;
}

extern "C" int pcst_gated_linear_bwd(const void* x, int dtype, int64_t M, int64_t D, const void* w_gate,
                                     const void* w_up, int64_t F, const void* b_gate, const void* b_up,
                                     int bias_f32, int act, const void* dh, void* dx, void* dw_gate,
                                     void* dw_up, int wgrad_f32, void* db_gate, void* db_up,
                                     void* workspace, void* stream) {
  if (int rc = check("gated_linear_bwd", dtype, M, D, F, act)) return rc;
  PCST_CHECK_ARG(dtype != kE4M3, "gated_linear_bwd: no gradients through e4m3 operands");
  PCST_CHECK_ARG((b_gate == nullptr) == (b_up == nullptr), "gated_linear_bwd: both biases or none");
  PCST_CHECK_ARG(M > 0, "gated_linear_bwd: no rows (the gradients of the weights are zero)");
  PCST_CHECK_ARG(x && w_gate && w_up && dh && workspace, "gated_linear_bwd: null pointer");
  const int es = elem(dtype);
  const Layout l = lay(workspace, dtype, M, D, F, true, true);
  gated::BwdCall c{};
  c.f.M = M;
  c.f.D = D;
  c.f.F = F;
  operands(c.f, l, x, w_gate, w_up, es, as_stream(stream));
  c.f.bg = b_gate;
  c.f.bu = b_up;
  c.f.bias_f32 = bias_f32;
  c.f.act = act;
  c.dh = dh;
  c.dgu = l.dgu;
  c.fpad = l.fpad;
  c.bpart = l.bpart;
  c.f.part = l.part;
  c.dx = dx;
  c.dwg = dw_gate;
  c.dwu = dw_up;
  c.dbg = db_gate;
  c.dbu = db_up;
  c.wgrad_f32 = wgrad_f32;
  c.bgrad_f32 = bias_f32;
  switch (dtype) {
    case kF32: return gated::bwd<EF32>(c, stream);
    case kBF16: return gated::bwd<EBF16>(c, stream);
    default: return gated::bwd<EF16>(c, stream);
  }
}
