// The matrix products of the gated linear layer (gated_linear.hip), for one operand type per
// translation unit.
//
//   forward     h[m, f] = act(g) * u,   g = sum_d x[m, d] Wg[f, d] + bg[f],   u likewise with Wu, bu
//   backward    dg = dh * u * act'(g),  du = dh * act(g)       (g and u recomputed, stored as [dg | du])
//               dx[m, d] = sum_f dg[m, f] Wg[f, d] + du[m, f] Wu[f, d]
//               dW[f, d] = sum_m dg[m, f] x[m, d]              (Wg; du for Wu)
//
// One tiled product serves all: out[m, n] = sum_k A(m, k) B(n, k), where either operand lies with k
// contiguous (x, W in the forward; [dg | du] in dx) or with its row index contiguous (W in dx; both
// operands of dW).  A work-group owns BM rows and two column blocks of BNH: Wg's and Wu's rows of the
// same features in the forward (so a lane holds g and u of the same element and the activation and the
// product need no exchange), neighbouring columns elsewhere.
//
// Staging: 128 bytes of k a stage (64 16-bit values, 32 floats, 128 e4m3), two stages, loaded from
// global memory straight into LDS while the other stage is multiplied.  The LDS image is linear in the
// order of the loading lanes; each lane picks the 16-byte piece it fetches (an XOR of the piece's index
// with bits of its row), so that the 16-byte fragment reads -- and the transposed 8-byte reads of
// operands whose rows are contiguous -- spread over the banks.  Loads past a tile's rows or past k are
// sent past the buffer's end and arrive as zeros, so ragged sizes take no other path.
//
// Outputs go to memory from the accumulators, 16 lanes side by side in a row: what counts is how many
// pieces a store falls into (16 rows a store: 1.9 M requests of 32 bytes for 60000 x 512 bf16, and twice
// the time).  In the forward, W's rows are dealt to the tiles so that a lane's tiles are consecutive
// features and 16 lanes a whole 128-byte line.
#pragma once
#include <type_traits>

#include "ops_types.h"

namespace pcst {
namespace gated {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __amdgpu_buffer_rsrc_t rsrc_t;
#define PCST_LDS __attribute__((address_space(3)))

enum { ACT_SILU = 0, ACT_GELU = 1, ACT_RELU = 2 };
enum { EPI_FWD = 0, EPI_BWD = 1, EPI_OUT = 2, EPI_RAW = 3 };  // RAW: g and u of a k split, fp32

constexpr int kRowB = 128;  // bytes of k per stage

struct GemmArgs {
  const char* a[2];   // row operand, per k segment
  const char* b0[2];  // column operand, per k segment: first (or only) matrix
  const char* b1[2];  // second matrix (forward / recompute)
  int64_t lda, ldb;   // bytes
  int64_t M;          // rows (per group)
  int N;              // columns of a column block's matrix
  int64_t K;          // per segment
  int tiles_m, tiles_n, ntiles, per_xcd;
  int splits;         // of k (row-contiguous operands only)
  int64_t kps;        // k per split
  int groups;         // independent products of one launch (dWg, dWu): group g's A starts a_group[g] bytes on
  int64_t a_group[2], o_split;  // bytes; elements from one split's output to the next one's
  void* out[2];       // per group
  int64_t ldo;        // elements
  const void *bg, *bu;
  int bias_f32;
  const void* dh;
  int64_t fpad;       // backward: du starts at column fpad of the [dg | du] rows
  float* bpart;       // backward: bias partials [row block, 2, N] or null
  const float *xs, *gs, *us;  // e4m3 scales
};

__device__ __forceinline__ rsrc_t make_rsrc(const char* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), (short)0, bytes > 0 ? bytes : 0, 0x00020000);
}

template <class E>
constexpr int elem_size() {
  return (int)sizeof(typename E::T);
}

// D += A B over the 16 bytes of k that a lane of each operand holds
template <class E>
__device__ __forceinline__ f32x4 mma16(i32x4 a, i32x4 b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mma16<EBF16>(i32x4 a, i32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma16<EF16>(i32x4 a, i32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma16<EF32>(i32x4 a, i32x4 b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__int_as_float(a[j]), __int_as_float(b[j]), c, 0, 0, 0);
  return c;
}
// e4m3: 32 bytes a lane, one 16x16x128 product (unit block scales); which k a byte is, is the same
// for both operands, which is all that the sum over k needs.  The unit adds the products of 8 bytes at 14
// bits below the binade of the largest (measured) and these sums in fp32: enough for a 16-bit result
// (2^-9 and 2^-11), not for a float one, so the 8-bit form has no float output.
__device__ __forceinline__ f32x4 mma32_e4m3(i32x4 a0, i32x4 a1, i32x4 b0, i32x4 b1, f32x4 c) {
  const i32x8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
  const i32x8 b = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
}

// ---- activations, of the hardware's exp2 and reciprocal (1 ulp of fp32 each).  fp32 outputs: the product g log2(e)
// is carried with its rounding error, exp2(p + d) = exp2(p) (1 + d ln 2), so that a sigmoid is off by a few 2^-24 at
// any g; expf and a division take five times the instructions (forward of 8000 x 256 x 512: 46.5 us, so 44.8).  16-bit types
// leave d out: |g| 2^-24, far below their rounding.
template <bool FAST>
__device__ __forceinline__ float sigmoid(float g) {
  constexpr float kLog2e = 1.44269504088896f, kLog2eLow = 1.92596299e-8f;  // their sum: log2(e) to 48 bits
  const float p = g * -kLog2e;
  float e = __builtin_amdgcn_exp2f(p);
  if (!FAST) {
    const float d = fmaf(g, -kLog2eLow, fmaf(g, -kLog2e, -p));
    // (inf stays inf: p is past 128 or not finite, d finite or NaN)
    e = fabsf(p) < 128.0f ? fmaf(e, d * 0.69314718f, e) : e;
  }
  return __builtin_amdgcn_rcpf(1.0f + e);
}
// 1 + erf(g / sqrt 2), e = exp(-g^2 / 2): Abramowitz and Stegun 7.1.26 (1.5e-7 absolute) for the 16-bit types
template <bool FAST>
__device__ __forceinline__ float gelu_cdf2(float g, float e) {
  if (!FAST) return 1.0f + erff(g * 0.70710678118654752f);
  const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(g), 0.3275911f * 0.70710678118654752f, 1.0f));
  const float c = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
  return g < 0.0f ? c * e : 2.0f - c * e;
}
template <bool FAST>
__device__ __forceinline__ float gauss(float g) {
  return FAST ? __builtin_amdgcn_exp2f(g * g * -0.72134752044448170f) : expf(-0.5f * g * g);
}
template <bool FAST, int ACT>
__device__ __forceinline__ float act_value(float g) {
  if (ACT == ACT_SILU) return g * sigmoid<FAST>(g);
  if (ACT == ACT_GELU) return 0.5f * g * gelu_cdf2<FAST>(g, FAST ? gauss<true>(g) : 0.0f);
  return g > 0.0f ? g : g * 0.0f;  // NaN stays NaN
}
template <bool FAST, int ACT>
__device__ __forceinline__ float act_grad(float g, float& value) {
  if (ACT == ACT_SILU) {
    const float e = sigmoid<FAST>(g);
    value = g * e;
    return e * (1.0f + g * (1.0f - e));
  }
  if (ACT == ACT_GELU) {
    const float e = gauss<FAST>(g), c = 0.5f * gelu_cdf2<FAST>(g, e);
    value = g * c;
    return fmaf(g * e, 0.3989422804014327f, c);
  }
  value = g > 0.0f ? g : g * 0.0f;
  return g > 0.0f ? 1.0f : g * 0.0f;
}

// ---- LDS images.  KC: row r holds 128 bytes of k; piece c of 16 bytes at position c ^ swz(r), so that the
// 16 lanes that read the same piece of 16 consecutive rows meet every bank once
__device__ __forceinline__ int swz_kc(int r) { return (r >> 1) & 7; }
// MN: row k holds W elements; 16-bit: transposed reads of rows k..k+3 (a group of 16 lanes) at 32
// bytes; fp32: 16 lanes read 64 bytes of one row, the four groups rows 4 apart
template <int ES, int CPR>
__device__ __forceinline__ int swz_mn(int k) {
  if (ES == 2) return (2 * ((k & 3) | (((k >> 3) & 1) << 2))) & (CPR - 1);
  return (4 * ((k >> 2) & 3)) & (CPR - 1);
}

// One operand's image of R rows (KC) or R columns (MN): R * 128 bytes either way.  DEAL > 1 (KC): row
// 16 t + j of each 16 * DEAL rows of the image is row DEAL j + t of the operand, so that lane j of a wave's
// DEAL tiles holds DEAL consecutive outputs.
template <class E, bool MN, int R, int DEAL, int NW>
struct Stage {
  static constexpr int ES = elem_size<E>();
  static constexpr int RB = R * ES;          // MN: bytes of one k row
  static constexpr int CPR = RB / 16;
  static constexpr int IT = R * kRowB / 1024 / NW;  // 1 KiB loads per wave
  static_assert(R * kRowB % (1024 * NW) == 0, "whole loads per wave");
  uint32_t off[IT];
  int piece[IT];  // KC: byte offset of the piece in its row (for the end of k)

  __device__ __forceinline__ void init(int wave, int lane, int64_t ld) {
#pragma unroll
    for (int j = 0; j < IT; ++j) {
      const int at = (wave + NW * j) * 1024 + lane * 16;
      if (MN) {
        const int k = at / RB, p = (at % RB) / 16;
        off[j] = (uint32_t)(k * ld + ((p ^ swz_mn<ES, CPR>(k)) * 16));
        piece[j] = 0;
      } else {
        const int r = at / kRowB, p = (at % kRowB) / 16;
        piece[j] = (p ^ swz_kc(r)) * 16;
        const int w = r % (16 * DEAL);
        off[j] = (uint32_t)((r - w + w % 16 * DEAL + w / 16) * ld + piece[j]);
      }
    }
  }
  // base: the tile's first byte at this stage's first k; bytes: up to the end of what may be read;
  // kleft: bytes of k left (KC)
  __device__ __forceinline__ void load(PCST_LDS char* img, const char* base, int bytes, int kleft, int wave) const {
    const rsrc_t r = make_rsrc(base, bytes);
#pragma unroll
    for (int j = 0; j < IT; ++j) {
      const uint32_t o = MN || piece[j] < kleft ? off[j] : 0x80000000u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (PCST_LDS void*)(img + (wave + NW * j) * 1024), 16, (int)o, 0, 0, 0);
    }
  }
};

// Fragment reads of one wave: T tiles of 16 rows from row r0 on; a lane gets 16 bytes of k of step ks
template <class E, bool MN, int R, int T>
struct Frag {
  static constexpr int ES = elem_size<E>();
  static constexpr int RB = R * ES, CPR = RB / 16;
  int at[MN ? T : 2];

  __device__ __forceinline__ void init(int r0, int lane) {
    const int l = lane & 15, g = lane >> 4;
    if (MN) {
#pragma unroll
      for (int t = 0; t < (MN ? T : 2); ++t) {
        if (ES == 2) {
          const int q = l >> 2, p = l & 3, k = 8 * g + q;
          const int c = (r0 + 16 * t) / 8 + (p >> 1);
          at[t] = k * RB + ((c ^ swz_mn<ES, CPR>(k)) * 16) + (p & 1) * 8;
        } else {
          const int k = 4 * g, c = (r0 + 16 * t) / 4 + (l >> 2);
          at[t] = k * RB + ((c ^ swz_mn<ES, CPR>(k)) * 16) + (l & 3) * 4;
        }
      }
    } else {
      const int r = r0 + l;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) at[ks] = r * kRowB + (((ks * 4 + g) ^ swz_kc(r)) * 16);
    }
  }
  __device__ __forceinline__ i32x4 read(const PCST_LDS char* img, int t, int ks) const {
    if (MN) {
      i32x4 v;
      if (ES == 2) {
        const PCST_LDS char* p = img + at[MN ? t : 0] + ks * 32 * RB;
        const i32x2 lo = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((PCST_LDS i16x4*)p));
        const i32x2 hi = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((PCST_LDS i16x4*)(p + 4 * RB)));
        v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = *(const PCST_LDS int*)(img + at[MN ? t : 0] + (ks * 16 + j) * RB);
      }
      return v;
    }
    return *(const PCST_LDS i32x4*)(img + at[MN ? 0 : ks] + t * 16 * kRowB);
  }
};

// N values of a vector of T or float from f on, n of them there; zeros elsewhere and for no vector
template <class T, int N>
__device__ __forceinline__ void load_bias(const void* b, int f32, int64_t f, int n, float (&v)[N]) {
  if (!b || n <= 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.0f;
  } else if (f32) {
    load_n<float, N>(static_cast<const float*>(b) + f, n, v);
  } else {
    load_n<T, N>(static_cast<const T*>(b) + f, n, v);
  }
}

// The gated epilogue of one wave: acc[0] (g) and acc[1] (u) of TM tiles of 16 rows, the lane's rows m + 16 i
// + 0..3, and TNH consecutive features from f on -> h, or [dg | du] and their column sums (before rounding)
template <class E, class O, int EPI, int ACT, int TM, int TNH>
__device__ __forceinline__ void gated_rows(const GemmArgs& g, const f32x4 (&acc)[2][TNH][TM], int64_t m0, int f,
                                           const float (&bg)[TNH], const float (&bu)[TNH], const float (&sg)[TNH],
                                           const float (&su)[TNH], float (&cg)[TNH], float (&cu)[TNH]) {
  constexpr int ES = elem_size<E>();
  constexpr bool FAST = ES < 4;
  const int n = g.N - f;
  // dh's rows are fetched AHEAD row tiles before their use, rows past the end as the last one: with each row's
  // load in front of its use, half of the epilogue is waiting
  typedef Vec<O, TNH> V;
  constexpr int AHEAD = EPI != EPI_BWD ? 1 : ES == 4 ? (TM < 2 ? TM : 2) : TM;
  typename V::V dv[AHEAD][4];
  auto fetch = [&](int i) {
    const O* dh = static_cast<const O*>(g.dh) + f;
    if (n >= TNH) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t m = m0 + 16 * i + r;
        dv[i % AHEAD][r] = *reinterpret_cast<const typename V::Any*>(dh + (m < g.M ? m : g.M - 1) * g.N);
      }
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t m = m0 + 16 * i + r;
#pragma unroll
        for (int t = 0; t < TNH; ++t) dv[i % AHEAD][r][t] = t < n ? dh[(m < g.M ? m : g.M - 1) * g.N + t] : (O)0.0f;
      }
    }
  };
  if (EPI == EPI_BWD) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) fetch(i);
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    float d[4][TNH];
    if (EPI == EPI_BWD) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < TNH; ++t) d[r][t] = (float)dv[i % AHEAD][r][t];
      if (i + AHEAD < TM) fetch(i + AHEAD);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t m = m0 + 16 * i + r;
      if (m >= g.M) continue;
      float gv[TNH], uv[TNH];
      const float xs = ES == 1 ? g.xs[m] : 1.0f;
#pragma unroll
      for (int t = 0; t < TNH; ++t) {
        gv[t] = acc[0][t][i][r];
        uv[t] = acc[1][t][i][r];
        if (ES == 1) {
          gv[t] *= xs * sg[t];
          uv[t] *= xs * su[t];
        }
        gv[t] += bg[t];
        uv[t] += bu[t];
      }
      if (EPI == EPI_FWD) {
        float o[TNH];
#pragma unroll
        for (int t = 0; t < TNH; ++t) o[t] = act_value<FAST, ACT>(gv[t]) * uv[t];
        if (n > 0) store_n<O, TNH>(static_cast<O*>(g.out[0]) + m * g.ldo + f, n, o);
      } else if (f < g.fpad) {
        float og[TNH], ou[TNH];
#pragma unroll
        for (int t = 0; t < TNH; ++t) {
          float v;
          const float da = act_grad<FAST, ACT>(gv[t], v);
          og[t] = t < n ? d[r][t] * uv[t] * da : 0.0f;  // the padding up to fpad is zero
          ou[t] = t < n ? d[r][t] * v : 0.0f;
          cg[t] += og[t];
          cu[t] += ou[t];
        }
        O* o = static_cast<O*>(g.out[0]) + m * g.ldo + f;
        store_n<O, TNH>(o, TNH, og);
        store_n<O, TNH>(o + g.fpad, TNH, ou);
      }
    }
  }
}

// E: operand type, O: output type, NMN / MMN: the column / row operand's row index is contiguous
template <class E, class O, bool NMN, bool MMN, int EPI, int ACT, int BM, int BNH, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, BM == 64 ? 4 : 2) void gemm_kernel(GemmArgs g) {
  constexpr int NW = WM * WN, TM = BM / WM / 16, TNH = BNH / WN / 16;
  constexpr int ES = elem_size<E>(), BKE = kRowB / ES;
  constexpr bool GATED = EPI != EPI_OUT;
  constexpr int NSEG = NMN && !MMN ? 2 : 1;  // k segments: dx sums over Wg, then over Wu
  constexpr bool LOOP = WM * WN == 4;  // several tiles a work-group
  static_assert(!GATED || !NMN, "the forward reads W with k contiguous");
  // one array per stage and operand, so that the compiler sees which loads a read has to wait for
  __shared__ __attribute__((aligned(1024))) char lds_a0[BM * kRowB], lds_a1[BM * kRowB];
  __shared__ __attribute__((aligned(1024))) char lds_b0[2 * BNH * kRowB], lds_b1[2 * BNH * kRowB];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;

  Stage<E, MMN, BM, 1, NW> sa;
  Stage<E, NMN, NMN ? 2 * BNH : BNH, NMN ? 1 : TNH, NW> sb;
  sa.init(wave, lane, g.lda);
  sb.init(wave, lane, g.ldb);
  Frag<E, MMN, BM, TM> fa;
  Frag<E, NMN, NMN ? 2 * BNH : BNH, TNH> fb[NMN ? 2 : 1];
  fa.init(wm * 16 * TM, lane);
  fb[0].init(wn * 16 * TNH, lane);
  if (NMN) fb[NMN ? 1 : 0].init(BNH + wn * 16 * TNH, lane);

  // LOOP: a work-group's tiles, one after the other; the next tile's first stage is loaded under the last
  // products of this one and its epilogue, which needs no LDS (the large tiles have no registers left for
  // it, and stages enough for the start of a tile not to matter).  Work-group L runs on XCD L % 8; an XCD's
  // tiles follow each other in blocks of 4 row tiles, so that what its work-groups read at a time is
  // shared in its L2.
  struct Tile {
    int64_t m0;
    int n0, tm, group, split, nk, total;
    int64_t klen;  // of a segment
    const char *pa[NSEG], *pb0[NSEG], *pb1[NSEG];  // per k segment, at its first k
    int ra, rb0, rb1;  // KC: bytes that may be read from there; MN: bytes of a row in front of the tile
  };
  auto decode = [&](int L, Tile& c) -> bool {
    const int idx = L >> 3;
    int t = (L & 7) * g.per_xcd + idx;
    if (idx >= g.per_xcd || t >= g.ntiles) return false;
    const int tiles_mn = g.tiles_m * g.tiles_n;
    const int gs = t / tiles_mn;
    t -= gs * tiles_mn;
    c.group = g.groups > 1 ? gs % g.groups : 0;
    c.split = g.groups > 1 ? gs / g.groups : gs;
    const int band = t / (4 * g.tiles_n), inb = t - band * 4 * g.tiles_n;
    const int bh = g.tiles_m - 4 * band < 4 ? g.tiles_m - 4 * band : 4;
    const int tn = inb / bh;
    c.tm = 4 * band + inb - tn * bh;
    c.m0 = (int64_t)c.tm * BM;
    c.n0 = tn * (GATED ? BNH : 2 * BNH);
    const int64_t kb = c.split * g.kps;
    c.klen = kb + g.kps < g.K ? g.kps : g.K - kb;
    c.nk = (int)((c.klen + BKE - 1) / BKE);
    c.total = c.nk * NSEG;
    const int64_t rows = g.M - c.m0 < BM ? g.M - c.m0 : BM;
    const int64_t cols = g.N - c.n0 < BNH ? g.N - c.n0 : BNH;
    const int64_t cols1 = GATED ? cols : g.N - c.n0 - BNH < BNH ? g.N - c.n0 - BNH : BNH;
    // (a tile's rows, and a stage's, are less than 2^31 bytes: the C entry's bounds)
    c.ra = MMN ? (int)(c.m0 * ES) : (int)(rows * g.lda - kb * ES);
    c.rb0 = NMN ? c.n0 * ES : (int)(cols * g.ldb - kb * ES);
    c.rb1 = (int)((cols1 > 0 ? cols1 : 0) * g.ldb - kb * ES);  // (NMN: not used)
#pragma unroll
    for (int q = 0; q < NSEG; ++q) {
      c.pa[q] = g.a[q] + g.a_group[c.group] + (MMN ? kb * g.lda + c.m0 * ES : c.m0 * g.lda + kb * ES);
      const int64_t ob = NMN ? kb * g.ldb + (int64_t)c.n0 * ES : (int64_t)c.n0 * g.ldb + kb * ES;
      c.pb0[q] = g.b0[q] + ob;
      c.pb1[q] = GATED ? g.b1[q] + ob : g.b0[q] + ob + (int64_t)BNH * g.ldb;
    }
    return true;
  };
  const int64_t step_a = MMN ? BKE * g.lda : kRowB, step_b = NMN ? BKE * g.ldb : kRowB;
  auto load = [&](const Tile& c, int it, PCST_LDS char* ia, PCST_LDS char* ib) {
    const int seg = NSEG > 1 && it >= c.nk ? 1 : 0;
    const int k = it - (seg ? c.nk : 0);
    const int64_t oa = k * step_a, ob = k * step_b;
    const int64_t left = c.klen - (int64_t)k * BKE;  // elements of k
    const int kn = left > BKE ? BKE : (int)left, kl = kn * ES;
    sa.load(ia, c.pa[seg] + oa, MMN ? kn * (int)g.lda - c.ra : c.ra - k * kRowB, kl, wave);
    sb.load(ib, c.pb0[seg] + ob, NMN ? kn * (int)g.ldb - c.rb0 : c.rb0 - k * kRowB, kl, wave);
    if (!NMN) sb.load(ib + BNH * kRowB, c.pb1[seg] + ob, c.rb1 - k * kRowB, kl, wave);
  };

  f32x4 acc[2][TNH][TM];
  auto compute = [&](const PCST_LDS char* ia, const PCST_LDS char* ib, auto&& prefetch) {
    if constexpr (ES == 1) {
      // a stage is one product deep; the fragments of two column tiles are read ahead of their products
      i32x4 a[2][TM], b[3][2];
      auto read_b = [&](int n) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) b[n % 3][ks] = fb[0].read(ib + n / TNH * BNH * kRowB, n % TNH, ks);
      };
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) a[ks][i] = fa.read(ia, i, ks);
      read_b(0);
      read_b(1);
      __builtin_amdgcn_sched_barrier(0);
      prefetch();
#pragma unroll
      for (int n = 0; n < 2 * TNH; ++n) {
        if (n + 2 < 2 * TNH) read_b(n + 2);
#pragma unroll
        for (int i = 0; i < TM; ++i)
          acc[n / TNH][n % TNH][i] = mma32_e4m3(a[0][i], a[1][i], b[n % 3][0], b[n % 3][1], acc[n / TNH][n % TNH][i]);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      // four groups (k step, column block) of TM * TNH products; a group's products run while the next
      // one's fragments are read
      i32x4 a[2][TM], b[2][TNH];
      auto read_a = [&](int ks) {
#pragma unroll
        for (int i = 0; i < TM; ++i) a[ks][i] = fa.read(ia, i, ks);
      };
      auto read_b = [&](int ks, int h) {
#pragma unroll
        for (int j = 0; j < TNH; ++j)
          b[h][j] = NMN ? fb[NMN ? h : 0].read(ib, j, ks) : fb[0].read(ib + h * BNH * kRowB, j, ks);
      };
      auto mma = [&](int ks, int h) {
#pragma unroll
        for (int j = 0; j < TNH; ++j)
#pragma unroll
          for (int i = 0; i < TM; ++i) acc[h][j][i] = GATED ? mma16<E>(a[ks][i], b[h][j], acc[h][j][i]) : mma16<E>(b[h][j], a[ks][i], acc[h][j][i]);
      };
      read_a(0);
      read_b(0, 0);
      read_b(0, 1);
      __builtin_amdgcn_sched_barrier(0);
      prefetch();  // the other stage's loads, behind this one's first reads and between the products
      mma(0, 0);
      read_a(1);
#pragma unroll
      for (int n = 0; n < TM * TNH; ++n) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // an MFMA,
        __builtin_amdgcn_sched_group_barrier(0x006, 6, 0);   // what prepares a load,
        __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);   // a load,
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);   // a fragment
      }
      __builtin_amdgcn_sched_barrier(0);
      read_b(1, 0);
      mma(0, 1);
      __builtin_amdgcn_sched_barrier(0);
      read_b(1, 1);
      mma(1, 0);
      __builtin_amdgcn_sched_barrier(0);
      mma(1, 1);
    }
  };

  PCST_LDS char* a0 = (PCST_LDS char*)lds_a0;
  PCST_LDS char* a1 = (PCST_LDS char*)lds_a1;
  PCST_LDS char* b0 = (PCST_LDS char*)lds_b0;
  PCST_LDS char* b1 = (PCST_LDS char*)lds_b1;
  auto next = [&]() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's loads of the stage
    __builtin_amdgcn_s_barrier();                     // everyone's; and the other stage has been read
    asm volatile("" ::: "memory");
  };
  // The same at the start of a tile, whose stage was loaded before the previous tile's stores: these stay
  // in flight.  kStores of them follow the loads where that tile was a whole one (`stores`); the counter
  // falls in order, so at kStores left, the loads are done.
  constexpr int kStores = EPI == EPI_FWD ? TM * 4 : EPI == EPI_RAW ? TM * 8 : TM * TNH * 2;
  auto first = [&](bool stores) {
    if (stores && LOOP && EPI != EPI_BWD)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kStores) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  Tile cur, nxt;
  int L = blockIdx.x;
  if (!decode(L, cur)) return;
  load(cur, 0, a0, b0);
  bool more = LOOP, stores = false;
  do {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < TNH; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[h][j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    // pairs of stages in one basic block: the accumulators stay in place
    first(stores);
    for (int it = 0; it + (LOOP ? 3 : 2) <= cur.total; it += 2) {
      compute(a0, b0, [&]() { load(cur, it + 1, a1, b1); });
      next();
      compute(a1, b1, [&]() { load(cur, it + 2, a0, b0); });  // past the last stage: fetches nothing
      next();
    }
    const int64_t m0 = cur.m0;
    const int n0 = cur.n0, tm = cur.tm;
    if (LOOP) {
      L += gridDim.x;
      more = decode(L, nxt);
    }
    if (cur.total & 1) {
      compute(a0, b0, []() {});
      if (LOOP) next();
      if (LOOP && more) load(nxt, 0, a0, b0);
    } else if (LOOP) {
      compute(a0, b0, [&]() { load(cur, cur.total - 1, a1, b1); });
      next();
      compute(a1, b1, [&]() { if (more) load(nxt, 0, a0, b0); });
    }

    asm volatile("" ::: "memory");  // the next tile's loads stay ahead of the stores
    stores = m0 + BM <= g.M && n0 + (GATED ? BNH : 2 * BNH) <= g.N;

  // ---- epilogue
  const int l = lane & 15, q = lane >> 4;
  if constexpr (EPI == EPI_RAW) {
    const int f = n0 + (wn * 16 + l) * TNH, n = g.N - f;
    float* out = static_cast<float*>(g.out[0]) + cur.split * g.o_split;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t m = m0 + wm * 16 * TM + 16 * i + 4 * q + r;
        if (m >= g.M || n <= 0) continue;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[TNH];
#pragma unroll
          for (int t = 0; t < TNH; ++t) v[t] = acc[h][t][i][r];
          store_n<float, TNH>(out + (h * g.M + m) * g.ldo + f, n, v);
        }
      }
  } else if constexpr (GATED) {
    // lane: row 4 q + r of each row tile, TNH consecutive features
    const int f = n0 + (wn * 16 + l) * TNH, n = g.N - f;
    float bg[TNH], bu[TNH], sg[TNH], su[TNH], cg[TNH], cu[TNH];
    load_bias<O, TNH>(g.bg, g.bias_f32, f, n, bg);
    load_bias<O, TNH>(g.bu, g.bias_f32, f, n, bu);
    if (ES == 1) {
      load_bias<float, TNH>(g.gs, 1, f, n, sg);
      load_bias<float, TNH>(g.us, 1, f, n, su);
    }
#pragma unroll
    for (int t = 0; t < TNH; ++t) cg[t] = cu[t] = 0.0f;
    gated_rows<E, O, EPI, ACT>(g, acc, m0 + wm * 16 * TM + 4 * q, f, bg, bu, sg, su, cg, cu);
    if (EPI == EPI_BWD && g.bpart) {  // column sums of the wave's rows, before rounding
      float* bp = g.bpart + ((int64_t)tm * WM + wm) * 2 * g.N + f;
#pragma unroll
      for (int t = 0; t < TNH; ++t) {
        cg[t] += __shfl_xor(cg[t], 16, 64);
        cg[t] += __shfl_xor(cg[t], 32, 64);
        cu[t] += __shfl_xor(cu[t], 16, 64);
        cu[t] += __shfl_xor(cu[t], 32, 64);
        if (q == 0 && t < n) {
          bp[t] = cg[t];
          bp[g.N + t] = cu[t];
        }
      }
    }
  } else {
    O* out = static_cast<O*>(g.out[cur.group]) + cur.split * g.o_split;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int64_t m = m0 + wm * 16 * TM + 16 * i + l;
      if (m >= g.M) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < TNH; ++j) {
          const int n = n0 + h * BNH + wn * 16 * TNH + (NMN ? 16 * j + 4 * q : q * 4 * TNH + 4 * j);
          if (n >= g.N) continue;
          const float v[4] = {acc[h][j][i][0], acc[h][j][i][1], acc[h][j][i][2], acc[h][j][i][3]};
          store_n<O, 4>(out + m * g.ldo + n, g.N - n, v);
        }
    }
  }
    if (LOOP) cur = nxt;
  } while (LOOP && more);
}

// ---- few rows (at most 128, see take_rows): the weights are read once, straight into the MFMA's registers.  A work-group owns
// 16 features of both matrices; its 8 waves split k and add up in LDS, in order.  Bound by reading the weights
// (and, at a handful of rows, by the launch: 1 x 1024 x 2816 bf16 4.8 us for 11.5 MB).  Rows may start at any element: no copies.
// 16 bytes of a row from `off` on, zeros past its end: where it ends inside, the row's last 16 moved down
template <class E>
__device__ __forceinline__ i32x4 piece16(const char* row, int64_t off, int64_t bytes) {
  typedef Vec<typename E::T, 16 / elem_size<E>()> V;
  if (off >= bytes) return i32x4{0, 0, 0, 0};
  const int64_t at = off + 16 <= bytes ? off : bytes - 16;
  if (at < 0) {  // (rows of less than 16 bytes)
    i32x4 v{0, 0, 0, 0};
#pragma unroll 1
    for (int b = 0; b < (int)bytes; ++b) v[b >> 2] |= (int)((uint32_t)(uint8_t)row[b] << (8 * (b & 3)));
    return v;
  }
  const i32x4 v = __builtin_bit_cast(i32x4, (typename V::V)*reinterpret_cast<const typename V::Any*>(row + at));
  const int n = (int)(off - at);  // bytes in front
  if (n == 0) return v;
  const unsigned __int128 w = __builtin_bit_cast(unsigned __int128, v) >> (8 * n);
  return __builtin_bit_cast(i32x4, w);
}

template <class E, class O, int ACT, int TM>
__global__ __launch_bounds__(512) void rows_kernel(GemmArgs g) {
  constexpr int ES = elem_size<E>(), P = ES == 1 ? 2 : 1, U = TM == 8 ? 1 : TM == 4 ? 2 : 4;  // pieces a product, products in flight
  __shared__ f32x4 red[8][2][TM][64];
  const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int f = blockIdx.x * 16 + l;
  const int64_t bytes = g.K * ES;
  const int steps = (int)((bytes + 64 * P - 1) / (64 * P)), per = (steps + 7) / 8;
  const int s0 = wave * per, s1 = s0 + per < steps ? s0 + per : steps;
  const int64_t fr = f < g.N ? f : g.N - 1;  // lanes past the end repeat the last row; their results are dropped
  const char *wg = g.b0[0] + fr * g.ldb, *wu = g.b1[0] + fr * g.ldb;
  const char* x[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) x[i] = g.a[0] + (16 * i + l < g.M ? 16 * i + l : g.M - 1) * g.lda;
  f32x4 acc[2][TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) acc[0][i] = acc[1][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  // UN steps at once; CHECK: a piece may end behind its row
  auto products = [&](int s, auto un, auto check) {
    constexpr int UN = decltype(un)::value;
    typedef Vec<typename E::T, 16 / ES> V;
    i32x4 a[UN][TM][P], b[UN][2][P];
    auto piece = [&](const char* row, int64_t off) {
      if constexpr (decltype(check)::value)
        return piece16<E>(row, off, bytes);
      else
        return __builtin_bit_cast(i32x4, (typename V::V)*reinterpret_cast<const typename V::Any*>(row + off));
    };
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int64_t off = ((int64_t)(s + u) * P + p) * 64 + q * 16;
        b[u][0][p] = piece(wg, off);
        b[u][1][p] = piece(wu, off);
#pragma unroll
        for (int i = 0; i < TM; ++i) a[u][i][p] = piece(x[i], off);
      }
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          if constexpr (ES == 1)
            acc[h][i] = mma32_e4m3(a[u][i][0], a[u][i][1], b[u][h][0], b[u][h][1], acc[h][i]);
          else
            acc[h][i] = mma16<E>(a[u][i][0], b[u][h][0], acc[h][i]);
        }
  };
  const int whole = (int)(bytes / (64 * P)) < s1 ? (int)(bytes / (64 * P)) : s1;
  int s = s0;
  for (; s + U <= whole; s += U) products(s, std::integral_constant<int, U>{}, std::false_type{});
  for (; s < whole; ++s) products(s, std::integral_constant<int, 1>{}, std::false_type{});
  if (s < s1) products(s, std::integral_constant<int, 1>{}, std::true_type{});
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < TM; ++i) red[wave][h][i][lane] = acc[h][i];
  __syncthreads();
  if (wave >= TM || f >= g.N) return;
  f32x4 gv = red[0][0][wave][lane], uv = red[0][1][wave][lane];
#pragma unroll
  for (int w = 1; w < 8; ++w) {
    gv += red[w][0][wave][lane];
    uv += red[w][1][wave][lane];
  }
  float bg[1], bu[1];
  load_bias<O, 1>(g.bg, g.bias_f32, f, 1, bg);
  load_bias<O, 1>(g.bu, g.bias_f32, f, 1, bu);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int64_t m = 16 * wave + 4 * q + r;
    if (m >= g.M) continue;
    float gr = gv[r], ur = uv[r];
    if (ES == 1) {
      gr *= g.xs[m] * g.gs[f];
      ur *= g.xs[m] * g.us[f];
    }
    gr += bg[0];
    ur += bu[0];
    static_cast<O*>(g.out[0])[m * g.ldo + f] = (O)(act_value<(ES < 4), ACT>(gr) * ur);
  }
}

// ---- narrow rows (K of at most 512 bytes, many rows): a work-group keeps 128 features of both matrices in
// LDS for its whole life, and each of its waves takes tiles of 64 or 32 rows by itself, straight from memory into
// registers: no barrier after the start, so that one wave's epilogue runs beside the other's products, and
// x is read once for every 128 features instead of W once for every 256 rows.  The next tile's rows are
// loaded as this one's are used for the last time.
constexpr int kNarrowF = 128, kNarrowBytes = 512;
// Rows of a wave's tile: what the registers hold of x beside the sums, of two groups of features where the outputs
// of one are made between the products of the next (x 256: 120000 rows 79 -> 75 us, 30000 27 -> 23 for the smaller
// tiles; x 128: no gain from it, so the larger tile).  Tiles go to the waves so that a SIMD's two waves differ
// where the number is no whole one (60000 x 256 x 512: 50 -> 42 us).
__host__ __device__ constexpr int narrow_rows_of(int64_t kbytes) { return kbytes <= 256 ? 64 : 32; }

// narrow_kernel's accesses: 2 features of a 16-bit matrix, addressed with 32 bits from the tile's first row (vo: the
// lane's offset; a row's is scalar).  FULL: both features and 4-byte accesses; else each value by itself, n of them.
template <class O, bool FULL>
__device__ __forceinline__ typename Vec<O, 2>::V narrow_load(rsrc_t from, int vo, int so, int n) {
  typename Vec<O, 2>::V v{};
  if (FULL) return __builtin_bit_cast(typename Vec<O, 2>::V, __builtin_amdgcn_raw_buffer_load_b32(from, vo, so, 0));
#pragma unroll
  for (int t = 0; t < 2; ++t)
    if (t < n) v[t] = __builtin_bit_cast(O, __builtin_amdgcn_raw_buffer_load_b16(from, vo + 2 * t, so, 0));
  return v;
}
template <class O, bool FULL>
__device__ __forceinline__ void narrow_store(typename Vec<O, 2>::V v, rsrc_t to, int vo, int so, int n) {
  if (FULL) {
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(int, v), to, vo, so, 0);
  } else {
#pragma unroll
    for (int t = 0; t < 2; ++t)
      if (t < n) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, (O)v[t]), to, vo + 2 * t, so, 0);
  }
}
// One row's 2 features (whose sums hold the biases): h, or dg and du `du` bytes on, with their column sums; n features
// are there, nz of them (with the padding of [dg | du]) are written
template <class O, int EPI, int ACT, bool FULL>
__device__ __forceinline__ void narrow_row(const float (&g)[2], const float (&u)[2], typename Vec<O, 2>::V d, rsrc_t to,
                                           int vo, int so, int du, int n, int nz, float (&cg)[2], float (&cu)[2]) {
  typename Vec<O, 2>::V o, p;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    if (EPI == EPI_FWD) {
      o[t] = (O)(act_value<true, ACT>(g[t]) * u[t]);
    } else {
      float v;
      const float da = act_grad<true, ACT>(g[t], v), dt = (float)d[t];
      const float og = FULL || t < n ? dt * u[t] * da : 0.0f, ou = FULL || t < n ? dt * v : 0.0f;
      cg[t] += og;
      cu[t] += ou;
      o[t] = (O)og;
      p[t] = (O)ou;
    }
  }
  narrow_store<O, FULL>(o, to, vo, so, EPI == EPI_FWD ? n : nz);
  if (EPI == EPI_BWD) narrow_store<O, FULL>(p, to, vo, so + du, nz);
}

template <class E, class O, int EPI, int ACT, int KS>
__global__ __launch_bounds__(512, 2) void narrow_kernel(GemmArgs g) {
  constexpr int ES = elem_size<E>(), kNarrowRows = narrow_rows_of(KS * 64), TM = kNarrowRows / 16, TNH = 2;
  constexpr int IM = KS / 2, SG = kNarrowF / 32;
  constexpr bool PIPED = KS == 8 && EPI == EPI_FWD;
  static_assert(KS == 8 || EPI == EPI_FWD, "the backward's: wider than 128");
  __shared__ __attribute__((aligned(1024))) char lds_w[IM * 2 * kNarrowF * kRowB];
  __shared__ float lds_b[2][kNarrowF];                                   // biases
  // tiles_n blocks of features x tiles_m groups of rows; an XCD's work-groups share row groups
  const int L = (blockIdx.x & 7) * g.per_xcd + (blockIdx.x >> 3);
  if (L >= g.ntiles) return;
  const int rg = L / g.tiles_n, n0 = (L - rg * g.tiles_n) * kNarrowF;
  const int tid = threadIdx.x, lane = tid & 63, l = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kb = (int)g.K * ES;
  PCST_LDS char* w = (PCST_LDS char*)lds_w;
  {
    Stage<E, false, kNarrowF, TNH, 8> sw;
    sw.init(wave, lane, g.ldb);
    const int rows = g.N - n0 < kNarrowF ? g.N - n0 : kNarrowF;
#pragma unroll
    for (int im = 0; im < IM; ++im)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        sw.load(w + (im * 2 + h) * kNarrowF * kRowB, (h ? g.b1[0] : g.b0[0]) + (int64_t)n0 * g.ldb + im * kRowB,
                (int)(rows * g.ldb) - im * kRowB, kb - im * kRowB, wave);
    if (tid < kNarrowF) {
      float v[1];
      load_bias<O, 1>(g.bg, g.bias_f32, n0 + tid, g.N - n0 - tid, v);
      lds_b[0][tid] = v[0];
      load_bias<O, 1>(g.bu, g.bias_f32, n0 + tid, g.N - n0 - tid, v);
      lds_b[1][tid] = v[0];
    }
  }
  Frag<E, false, kNarrowF, TNH> fb;
  fb.init(0, lane);

  // of the two waves of a SIMD, one goes first through its products: they come apart, and one's epilogue
  // runs beside the other's products
  const bool ahead = wave < 4;
  i32x4 x[TM][KS];
  typedef typename Vec<O, 2>::V V2;
  constexpr int NP = TM * 4;  // a lane's rows of a tile
  float cg[SG][TNH], cu[SG][TNH];  // column sums of the wave's rows, by group of features
#pragma unroll
  for (int i = 0; i < SG; ++i)
#pragma unroll
    for (int t = 0; t < TNH; ++t) cg[i][t] = cu[i][t] = 0.0f;
  // 4-byte accesses of pairs of features: an even number of them, rows on 4-byte boundaries; pairs past the end are
  // sent past the buffer's (dh's are zeros there, as the sums are, and so is what is written up to fpad)
  const bool pairs = (g.N & 1) == 0 && (((uintptr_t)g.out[0] | (EPI == EPI_BWD ? (uintptr_t)g.dh : 0)) & 3) == 0;
  const int pitch = (int)g.ldo * 2, pd = g.N * 2, du = (int)g.fpad * 2, limit = EPI == EPI_FWD ? g.N : (int)g.fpad;
  auto pair_at = [&](int sgi, int row, int end) {
    const int f = n0 + sgi * 32 + l * TNH;
    return f < end ? 4 * q * row + f * 2 : (int)0x80000000;
  };
  const int step = g.tiles_m * 8, tiles = (int)((g.M + kNarrowRows - 1) / kNarrowRows);
  int tile = wave * g.tiles_m + rg;
  auto tile_rsrc = [&](int t) {
    const int64_t m0 = (int64_t)t * kNarrowRows, rows = g.M - m0 < kNarrowRows ? g.M - m0 : kNarrowRows;
    return make_rsrc(g.a[0] + m0 * g.lda, t < tiles ? (int)(rows * g.lda) : 0);  // past the last tile: fetches nothing
  };
  auto load_x = [&](rsrc_t r, int i, int ks) {
    const int o = ks * 64 + q * 16 < kb ? (int)((16 * i + l) * g.lda) + ks * 64 + q * 16 : (int)0x80000000;
    return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, o, 0, 0));
  };
  {
    const rsrc_t r = tile_rsrc(tile);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < TM; ++i) x[i][ks] = load_x(r, i, ks);
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");

  // A whole tile: a group's outputs are made between the products of the next one, a few instructions behind
  // each, so that the matrix unit and the others work at the same time in every wave.
  auto piped = [&](rsrc_t ro, rsrc_t rn) {
    if constexpr (PIPED) {
    f32x4 acc[2][2][TNH][TM];
    auto piece = [&](int sgi, int p) {
      const int i = p / 4, e = p % 4;
      const float gv[2] = {acc[sgi & 1][0][0][i][e], acc[sgi & 1][0][1][i][e]};
      const float uv[2] = {acc[sgi & 1][1][0][i][e], acc[sgi & 1][1][1][i][e]};
      narrow_row<O, EPI, ACT, true>(gv, uv, V2{}, ro, pair_at(sgi, pitch, limit), (16 * i + e) * pitch, du, 2, 2, cg[sgi],
                                    cu[sgi]);
    };
#pragma unroll
    for (int sgi = 0; sgi < SG; ++sgi) {
      const PCST_LDS char* ws = w + sgi * 32 * kRowB;
      i32x4 b[2][2][TNH];
      auto read = [&](int ks) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < TNH; ++t) b[ks & 1][h][t] = fb.read(ws + ((ks >> 1) * 2 + h) * kNarrowF * kRowB, t, ks & 1);
      };
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < TNH; ++t) {
          const float v = lds_b[h][sgi * 32 + l * TNH + t];
#pragma unroll
          for (int i = 0; i < TM; ++i) acc[sgi & 1][h][t][i] = f32x4{v, v, v, v};
        }
      read(0);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (ks + 1 < KS) read(ks + 1);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < TNH; ++t)
#pragma unroll
            for (int i = 0; i < TM; ++i)
              acc[sgi & 1][h][t][i] = mma16<E>(x[i][ks], b[ks & 1][h][t], acc[sgi & 1][h][t][i]);
        if (sgi) {
#pragma unroll
          for (int p = ks * NP / KS; p < (ks + 1) * NP / KS; ++p) piece(sgi - 1, p);
        }
        if (sgi == SG - 1) {
#pragma unroll
          for (int i = 0; i < TM; ++i) x[i][ks] = load_x(rn, i, ks);
        }
#pragma unroll
        for (int n = 0; n < 4 * TM; ++n) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                        // an MFMA,
          __builtin_amdgcn_sched_group_barrier(0x002, ACT == ACT_GELU ? 6 : 3, 0);  // what runs beside it
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) piece(SG - 1, p);
    }
  };

  for (; tile < tiles; tile += step) {
    const int64_t mt = (int64_t)tile * kNarrowRows;
    const rsrc_t ro = make_rsrc(static_cast<char*>(g.out[0]) + mt * g.ldo * 2, 0x7fffffff);
    const rsrc_t rd = make_rsrc(static_cast<const char*>(g.dh) + mt * g.N * 2, 0x7fffffff);
    const bool full = pairs && mt + kNarrowRows <= g.M;
    const rsrc_t rn = tile_rsrc(tile + step);
    auto group = [&](int sgi, auto last) {
      // the sums start at the biases
      const int c = sgi * 32 + l * TNH;
      f32x4 acc[2][TNH][TM], c0[2][TNH];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < TNH; ++t) {
          const float v = lds_b[h][c + t];
          c0[h][t] = f32x4{v, v, v, v};
        }
      const int rows = (int)(g.M - mt < kNarrowRows ? g.M - mt : kNarrowRows) - 4 * q, f = n0 + c, n = g.N - f;
      V2 d[EPI == EPI_BWD ? NP : 1];
      if (EPI == EPI_BWD) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const int row = 16 * (p / 4) + p % 4;
          V2& v = d[EPI == EPI_BWD ? p : 0];
          if (full) v = narrow_load<O, true>(rd, pair_at(sgi, pd, g.N), row * pd, 2);
          else v = narrow_load<O, false>(rd, 4 * q * pd + f * 2, row * pd, row < rows ? n : 0);
        }
      }
      const PCST_LDS char* ws = w + sgi * 32 * kRowB;
      i32x4 b[2][2][TNH];
      auto read = [&](int ks) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < TNH; ++t) b[ks & 1][h][t] = fb.read(ws + ((ks >> 1) * 2 + h) * kNarrowF * kRowB, t, ks & 1);
      };
      {
        read(0);
        if (ahead) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if (ks + 1 < KS) read(ks + 1);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int t = 0; t < TNH; ++t)
#pragma unroll
              for (int i = 0; i < TM; ++i) acc[h][t][i] = mma16<E>(x[i][ks], b[ks & 1][h][t], ks ? acc[h][t][i] : c0[h][t]);
          if constexpr (decltype(last)::value) {
#pragma unroll
            for (int i = 0; i < TM; ++i) x[i][ks] = load_x(rn, i, ks);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
      // (rows past the end: nothing is written, and dh's zeros add nothing to the column sums)
      auto rows_out = [&](auto whole_rows) {
        constexpr bool FULL = decltype(whole_rows)::value;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const int i = p / 4, row = 16 * i + p % 4;
          const float gv[2] = {acc[0][0][i][p % 4], acc[0][1][i][p % 4]}, uv[2] = {acc[1][0][i][p % 4], acc[1][1][i][p % 4]};
          if (FULL || row < rows)
            narrow_row<O, EPI, ACT, FULL>(gv, uv, d[EPI == EPI_BWD ? p : 0], ro,
                                          FULL ? pair_at(sgi, pitch, limit) : 4 * q * pitch + f * 2, row * pitch, du, n,
                                          limit - f, cg[sgi], cu[sgi]);
        }
      };
      if (!PIPED && full) rows_out(std::true_type{});
      else rows_out(std::false_type{});
    };
    if (PIPED && full) {
      piped(ro, rn);
      continue;
    }
#pragma unroll
    for (int sgi = 0; sgi < SG - 1; ++sgi) group(sgi, std::false_type{});
    group(SG - 1, std::true_type{});
  }
  if (EPI == EPI_BWD && g.bpart) {
    float* bp = g.bpart + ((int64_t)rg * 8 + wave) * 2 * g.N + n0;
#pragma unroll
    for (int sgi = 0; sgi < SG; ++sgi)
#pragma unroll
      for (int t = 0; t < TNH; ++t) {
        float a = cg[sgi][t], b = cu[sgi][t];
        a += __shfl_xor(a, 16, 64);
        a += __shfl_xor(a, 32, 64);
        b += __shfl_xor(b, 16, 64);
        b += __shfl_xor(b, 32, 64);
        const int c = sgi * 32 + l * TNH + t;
        if (q == 0 && n0 + c < g.N) {
          bp[c] = a;
          bp[g.N + c] = b;
        }
      }
  }
}

// ---- host side of one operand type
struct FwdCall {
  const void *x, *wg, *wu;
  int64_t M, D, F, ldx, ldw;  // pitches in bytes, 16-byte multiples, bases 16-byte aligned
  const void *bg, *bu;
  int bias_f32, act, out_type;
  const float *xs, *gs, *us;
  float* part;  // partial sums of split products
  void* h;
};
struct BwdCall {
  FwdCall f;
  const void* dh;
  void* dgu;       // [M, 2 * fpad]
  int64_t fpad;
  float* bpart;
  void *dx, *dwg, *dwu, *dbg, *dbu;
  int wgrad_f32, bgrad_f32;
};

// ---- which tiles, and over how many splits of k
// Tiles of 256 x 2*128, 128 x 2*64 and 64 x 2*32; 1, 2 and 4 work-groups of them run on a CU.  With the device full
// the largest reach 1.17 PFLOP/s (8192 x 4096 x 8192 bf16, 936 us; a plain product of this size in the library 1.33)
// and 2.2 to 2.4 in e4m3 (465 to 505 us; 2.85), the matrix units busy in 61 % of the cycles.  What bounds them is
// power: waves that take turns at reading and multiplying, over half-length stages, kept them busy in 69 % of
// 11 % fewer cycles, and the clock fell from 1.83 to 1.67 GHz (912 us, shorter sums slower).  float: 138 TFLOP/s of 152.
// The time of a
// launch is estimated as rounds of work-groups x (stages x a stage's time + a tile's start and end), both
// measured with the device full (us, 16-bit: 8192 x 4096 x 8192; start and end: 60000 x 512 with k = 64 .. 512);
// a round that leaves CUs with fewer work-groups is faster by that, down to the latency of a load.  Splitting
// k costs a launch and the partial sums' way through memory.
struct Tiling {
  int bm, bnh, wm, wn, per_cu;
  double stage[3], ends;  // stage: 16-bit, float, e4m3
};
constexpr Tiling kTilings[3] = {{256, 128, 4, 2, 1, {1.8, 7.8, 2.0}, 6.0},
                                {128, 64, 2, 2, 2, {0.98, 3.9, 1.1}, 3.7},
                                {64, 32, 2, 2, 4, {0.75, 2.05, 0.9}, 2.0}};
constexpr double kStageMin = 0.8, kSplitUs = 5.0, kBytesPerUs = 8e6;

struct Plan {
  int tiling, splits;
  int64_t kps;
  double us;
};

// rows x cols outputs of `groups` products with `segs` sums of K; wide: a tile is 2 * bnh columns (else the
// two blocks are Wg's and Wu's); outputs: fp32 values of one partial
inline Plan plan(int64_t rows, int64_t cols, int64_t K, int segs, int groups, bool wide, int es, int64_t outputs) {
  Plan best{0, 1, K, 1e300};
  const int64_t bke = kRowB / es, stages = cdiv(K, bke);
  for (int c = 0; c < 3; ++c) {
    const Tiling& t = kTilings[c];
    const double ts = t.stage[es == 4 ? 1 : es == 1 ? 2 : 0];
    const int64_t tiles = cdiv(rows, t.bm) * cdiv(cols, wide ? 2 * t.bnh : t.bnh) * groups;
    for (int64_t s = 1; s <= 64 && s <= stages; s *= 2) {
      if (s > 1 && (c == 0 || tiles * (s / 2) >= 256 * t.per_cu)) break;  // the device is full without
      const int64_t per = cdiv(stages, s), n = tiles * cdiv(stages, per), slots = 256 * t.per_cu;
      const double part = std::max(std::min(kStageMin, ts), ts * (double)cdiv(n % slots, 256) / t.per_cu);
      const double us = (double)(n / slots) * ((double)(per * segs) * ts + t.ends) +
                        (n % slots ? (double)(per * segs) * part + t.ends : 0.0) +
                        (s > 1 ? kSplitUs + 8.0 * (double)outputs * (double)s / kBytesPerUs : 0.0);
      if (us < best.us) best = Plan{c, (int)cdiv(stages, per), s > 1 ? per * bke : K, us};
    }
  }
  return best;
}
inline Plan plan_gated(int64_t M, int64_t D, int64_t F, int es) { return plan(M, F, D, 1, 1, false, es, 2 * M * F); }
// narrow rows (16 bits): taken where 5 us and 1.13 (k of 256 bytes: 1.57) for each tile of a CU, as measured (us;
// forward of 60000 x 512: D = 128 28 against 40 for the tiles above, 256 42 against 55), are less than the tiles'
// estimate.  The backward's form waits for dh and x longer, and both write twice as much: 20 us and 1.93 for each
// tile against 1.7 times the estimate (x 256 x 512 out of HBM: 30000 rows 49 against 46, 60000 76 against 88, 120000
// 134 against 180); up to 128 columns no gain.
inline int64_t narrow_groups(int64_t M, int64_t F, int64_t kbytes) {
  return std::max<int64_t>(1, std::min<int64_t>(256 / cdiv(F, kNarrowF), cdiv(cdiv(M, narrow_rows_of(kbytes)), 8)));
}
inline bool take_narrow(int64_t M, int64_t D, int64_t F, bool bwd) {
  const int64_t kbytes = 2 * D;
  if (kbytes > kNarrowBytes || cdiv(F, kNarrowF) > 256 || (bwd && kbytes <= 256)) return false;
  const int64_t each = cdiv(cdiv(M, narrow_rows_of(kbytes)), narrow_groups(M, F, kbytes));
  const double tiles = plan_gated(M, D, F, 2).us;
  return bwd ? 20.0 + 1.93 * (double)each < 1.7 * tiles : 5.0 + (kbytes <= 256 ? 1.57 : 1.13) * (double)each < tiles;
}
// few rows: always up to 16 (no workspace to ask for), up to 128 where 3.5 us and 0.45 + 0.19 for each 16 rows of x
// per 512 bytes of k and 256 work-groups are less than the tiles' estimate, the launch that adds their splits
// and the copies of ragged rows.  Measured (us, bf16): 1024 x 2816: 16 rows 5.5 against 9.3 for tiles, 64 8.6 against
// 13.9, 4096 x 1000: 13.1 against 14.6, 24.3 against 14.6; 1001 x 3000: 15.6 against 28 at 64 rows.
constexpr int kRowsFew = 16, kRowsMax = 128;
inline bool take_rows(int64_t M, int64_t D, int64_t F, int es) {
  if (M <= kRowsFew || M > kRowsMax) return M <= kRowsFew;
  const double tm = M <= 32 ? 2.0 : M <= 64 ? 4.0 : es == 4 ? 12.0 : 10.0;  // (from 65 rows on one work-group a CU)
  const double rows = 3.5 + (0.45 + 0.19 * tm) * (double)cdiv(D * es, 512) * std::max(1.0, (double)F / 4096.0);
  return rows < plan_gated(M, D, F, es).us + 2.5 + (D * es % 16 ? 12.0 : 0.0);
}
inline Plan plan_dx(int64_t M, int64_t D, int64_t F, int es) { return plan(M, D, F, 2, 1, true, es, M * D); }
inline Plan plan_dw(int64_t M, int64_t D, int64_t F, int es) { return plan(F, D, M, 1, 2, true, es, 2 * F * D); }

// floats of partial sums that a call needs, one product at a time
inline int64_t part_floats(int64_t M, int64_t D, int64_t F, int es, bool bwd) {
  auto need = [](const Plan& p, int64_t outputs) { return p.splits > 1 ? p.splits * outputs : 0; };
  int64_t n = need(plan_gated(M, D, F, es), 2 * M * F);
  if (bwd) {
    n = std::max(n, need(plan_dx(M, D, F, es), M * D));
    n = std::max(n, need(plan_dw(M, D, F, es), 2 * F * D));
  }
  return n;
}
// rows of bias partials: one for each wave's rows of a tile, or for 16 rows where k is split (few rows a
// work-group: the splits' values are fetched one row after the other)
constexpr int kFinishRows = 16;
inline int64_t bias_parts(int64_t M, int64_t D, int64_t F, int es, const Plan& p) {
  if (es == 2 && take_narrow(M, D, F, true)) return 8 * narrow_groups(M, F, D * es);  // its waves' rows
  return p.splits > 1 ? cdiv(M, kFinishRows) : cdiv(M, kTilings[p.tiling].bm) * kTilings[p.tiling].wm;
}

template <class E>
int fwd(const FwdCall& c, void* stream);
template <class E>
int bwd(const BwdCall& c, void* stream);

#ifdef PCST_GATED_IMPL
template <class E, class O, bool NMN, bool MMN, int EPI, int ACT, int C>
int launch_tiling(GemmArgs& g, hipStream_t s) {
  constexpr Tiling t = kTilings[C];
  const int64_t tm = cdiv(g.M, t.bm), tn = cdiv(g.N, EPI == EPI_OUT ? 2 * t.bnh : t.bnh), n = tm * tn * g.groups * g.splits;
  PCST_CHECK_ARG(n < (1ll << 30), "gated_linear: too many tiles");
  g.tiles_m = (int)tm;
  g.tiles_n = (int)tn;
  g.ntiles = (int)n;
  g.per_xcd = (int)cdiv(n, 8);
  // the smaller tiles: as many work-groups as run at a time
  const unsigned grid = (unsigned)(C == 0 ? g.per_xcd * 8 : std::min<int64_t>(g.per_xcd * 8, 256 * t.per_cu));
  hipLaunchKernelGGL((gemm_kernel<E, O, NMN, MMN, EPI, ACT, t.bm, t.bnh, t.wm, t.wn>), dim3(grid),
                     dim3(64 * t.wm * t.wn), 0, s, g);
  PCST_LAUNCH_CHECK("gated_linear");
  return PCST_OK;
}
template <class E, class O, bool NMN, bool MMN, int EPI, int ACT>
int launch(GemmArgs& g, int tiling, hipStream_t s) {
  if (tiling == 0 && EPI != EPI_RAW) return launch_tiling<E, O, NMN, MMN, EPI, ACT, EPI == EPI_RAW ? 1 : 0>(g, s);
  return tiling == 1 ? launch_tiling<E, O, NMN, MMN, EPI, ACT, 1>(g, s) : launch_tiling<E, O, NMN, MMN, EPI, ACT, 2>(g, s);
}
template <class E, class O, int EPI, int ACT>
int launch_narrow(GemmArgs& g, hipStream_t s) {
  g.tiles_n = (int)cdiv(g.N, kNarrowF);
  g.tiles_m = (int)narrow_groups(g.M, g.N, g.K * elem_size<E>());
  g.ntiles = g.tiles_n * g.tiles_m;
  g.per_xcd = (int)cdiv(g.ntiles, 8);
  const dim3 grid((unsigned)(g.per_xcd * 8));
  if constexpr (EPI == EPI_FWD) {
    if (g.K * elem_size<E>() <= 256) {
      hipLaunchKernelGGL((narrow_kernel<E, O, EPI, ACT, 4>), grid, dim3(512), 0, s, g);
      PCST_LAUNCH_CHECK("gated_linear");
      return PCST_OK;
    }
  }
  hipLaunchKernelGGL((narrow_kernel<E, O, EPI, ACT, 8>), grid, dim3(512), 0, s, g);
  PCST_LAUNCH_CHECK("gated_linear");
  return PCST_OK;
}
template <class E, class O, int EPI>
int launch_act(GemmArgs& g, int tiling, int act, hipStream_t s) {
  return act == ACT_SILU   ? launch<E, O, false, false, EPI, ACT_SILU>(g, tiling, s)
         : act == ACT_GELU ? launch<E, O, false, false, EPI, ACT_GELU>(g, tiling, s)
                           : launch<E, O, false, false, EPI, ACT_RELU>(g, tiling, s);
}

// ---- the gated epilogues behind a split k: the splits added in order, then as above.  A work-group takes 64
// features of kFinishRows rows.
struct FinishArgs {
  const float* part;  // [splits, 2, M, F]
  int splits;
  int64_t M;
  int F;
  const void *bg, *bu;
  int bias_f32;
  const float *xs, *gs, *us;
  const void* dh;
  void* out;
  int64_t ldo, fpad;
  float* bpart;
};
template <class E, class O, int EPI, int ACT>
__global__ __launch_bounds__(256) void finish_kernel(FinishArgs a) {
  constexpr bool FAST = elem_size<E>() < 4;
  __shared__ float red[2][4][64];
  const int c = threadIdx.x & 63, w = threadIdx.x >> 6, f = blockIdx.x * 64 + c;
  const int64_t m0 = (int64_t)blockIdx.y * kFinishRows, n = a.M * a.F;
  const bool in = f < a.F;
  float bg[1] = {0.f}, bu[1] = {0.f}, cg = 0.0f, cu = 0.0f;
  if (in) {
    load_bias<O, 1>(a.bg, a.bias_f32, f, 1, bg);
    load_bias<O, 1>(a.bu, a.bias_f32, f, 1, bu);
  }
  // a wave's rows and eight splits at a time in flight, whatever their number: past the end the last one again, unused
  constexpr int R = kFinishRows / 4;
  float gs[R], us[R];
  const float* p[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int64_t m = m0 + w + 4 * j;
    p[j] = a.part + (m < a.M ? m : a.M - 1) * a.F + (in ? f : a.F - 1);
    gs[j] = us[j] = 0.0f;
  }
  for (int k0 = 0; k0 < a.splits; k0 += 8) {
    float v[8][R][2];
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int j = 0; j < R; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) v[k][j][h] = p[j][(2 * (int64_t)(k0 + k < a.splits ? k0 + k : a.splits - 1) + h) * n];
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int j = 0; j < R; ++j) {
        gs[j] += k0 + k < a.splits ? v[k][j][0] : 0.0f;
        us[j] += k0 + k < a.splits ? v[k][j][1] : 0.0f;
      }
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int64_t m = m0 + w + 4 * j;
    if (m >= a.M) continue;
    float g = gs[j], u = us[j];
    if (in) {
      if (elem_size<E>() == 1) {
        g *= a.xs[m] * a.gs[f];
        u *= a.xs[m] * a.us[f];
      }
      g += bg[0];
      u += bu[0];
    }
    if (EPI == EPI_FWD) {
      if (in) static_cast<O*>(a.out)[m * a.ldo + f] = (O)(act_value<FAST, ACT>(g) * u);
    } else {  // (f < fpad: a multiple of 64)
      float v, og = 0.0f, ou = 0.0f;
      const float da = act_grad<FAST, ACT>(g, v);
      if (in) {
        const float d = (float)static_cast<const O*>(a.dh)[m * a.F + f];
        og = d * u * da;
        ou = d * v;
        cg += og;
        cu += ou;
      }
      static_cast<O*>(a.out)[m * a.ldo + f] = (O)og;
      static_cast<O*>(a.out)[m * a.ldo + a.fpad + f] = (O)ou;
    }
  }
  if (EPI == EPI_BWD && a.bpart) {
    red[0][w][c] = cg;
    red[1][w][c] = cu;
    __syncthreads();
    if (w < 2 && in)
      a.bpart[((int64_t)blockIdx.y * 2 + w) * a.F + f] = red[w][0][c] + red[w][1][c] + red[w][2][c] + red[w][3][c];
  }
}
template <class E, class O, int EPI>
int launch_finish(const FinishArgs& a, int act, hipStream_t s) {
  const dim3 grid((unsigned)cdiv(a.F, 64), (unsigned)cdiv(a.M, kFinishRows));
  if (act == ACT_SILU) hipLaunchKernelGGL((finish_kernel<E, O, EPI, ACT_SILU>), grid, dim3(256), 0, s, a);
  else if (act == ACT_GELU) hipLaunchKernelGGL((finish_kernel<E, O, EPI, ACT_GELU>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((finish_kernel<E, O, EPI, ACT_RELU>), grid, dim3(256), 0, s, a);
  PCST_LAUNCH_CHECK("gated_linear");
  return PCST_OK;
}

// the forward (EPI_FWD, into out) or the recomputing backward (EPI_BWD, into [dg | du])
template <class E, class O, int EPI>
int run_gated(GemmArgs& g, const Plan& p, int act, float* part, hipStream_t s) {
  if constexpr (elem_size<E>() == 2) {
    if (take_narrow(g.M, g.K, g.N, EPI == EPI_BWD))
      return act == ACT_SILU   ? launch_narrow<E, O, EPI, ACT_SILU>(g, s)
             : act == ACT_GELU ? launch_narrow<E, O, EPI, ACT_GELU>(g, s)
                               : launch_narrow<E, O, EPI, ACT_RELU>(g, s);
  }
  if (p.splits == 1) return launch_act<E, O, EPI>(g, p.tiling, act, s);
  const FinishArgs a{part,  p.splits, g.M, g.N, g.bg, g.bu, g.bias_f32, g.xs, g.gs, g.us, g.dh, g.out[0], g.ldo, g.fpad,
                     g.bpart};
  g.splits = p.splits;
  g.kps = p.kps;
  g.out[0] = part;
  g.ldo = g.N;
  g.o_split = 2 * g.M * g.N;
  if (int rc = launch<E, float, false, false, EPI_RAW, 0>(g, p.tiling, s)) return rc;
  return launch_finish<E, O, EPI>(a, act, s);
}

inline GemmArgs fwd_args(const FwdCall& c) {
  GemmArgs g{};
  g.a[0] = static_cast<const char*>(c.x);
  g.b0[0] = static_cast<const char*>(c.wg);
  g.b1[0] = static_cast<const char*>(c.wu);
  g.lda = c.ldx;
  g.ldb = c.ldw;
  g.M = c.M;
  g.N = (int)c.F;
  g.K = g.kps = c.D;
  g.splits = g.groups = 1;
  g.bg = c.bg;
  g.bu = c.bu;
  g.bias_f32 = c.bias_f32;
  g.xs = c.xs;
  g.gs = c.gs;
  g.us = c.us;
  return g;
}

template <class E, class O, int ACT>
int launch_rows(const GemmArgs& g, hipStream_t s) {
  const dim3 grid((unsigned)cdiv(g.N, 16));
  if (g.M <= 16) hipLaunchKernelGGL((rows_kernel<E, O, ACT, 1>), grid, dim3(512), 0, s, g);
  else if (g.M <= 32) hipLaunchKernelGGL((rows_kernel<E, O, ACT, 2>), grid, dim3(512), 0, s, g);
  else if (g.M <= 64) hipLaunchKernelGGL((rows_kernel<E, O, ACT, 4>), grid, dim3(512), 0, s, g);
  else hipLaunchKernelGGL((rows_kernel<E, O, ACT, 8>), grid, dim3(512), 0, s, g);
  PCST_LAUNCH_CHECK("gated_linear");
  return PCST_OK;
}

template <class E, class O>
int fwd_out(const FwdCall& c, hipStream_t s) {
  GemmArgs g = fwd_args(c);
  g.out[0] = c.h;
  g.ldo = c.F;
  if (take_rows(c.M, c.D, c.F, elem_size<E>()))
    return c.act == ACT_SILU   ? launch_rows<E, O, ACT_SILU>(g, s)
           : c.act == ACT_GELU ? launch_rows<E, O, ACT_GELU>(g, s)
                               : launch_rows<E, O, ACT_RELU>(g, s);
  return run_gated<E, O, EPI_FWD>(g, plan_gated(c.M, c.D, c.F, elem_size<E>()), c.act, c.part, s);
}

// Bias gradients from the row blocks' partials [parts, 2, F]: 16 columns a work-group, 16 slices of the parts
struct BiasArgs {
  const float* part;
  int F, parts, f32;
  void *dbg, *dbu;
};
template <class T>
__device__ __forceinline__ void bias_columns(const BiasArgs& b, int block) {
  __shared__ double red[16][17];
  const int c = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int f = block * 16 + c;  // of 2 F
  double s = 0.0;
  if (f < 2 * b.F) {
    for (int p0 = q; p0 < b.parts; p0 += 16 * 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = b.part[(int64_t)(p0 + 16 * k < b.parts ? p0 + 16 * k : p0) * 2 * b.F + f];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += p0 + 16 * k < b.parts ? (double)v[k] : 0.0;
    }
  }
  red[q][c] = s;
  __syncthreads();
  if (q == 0 && f < 2 * b.F) {
    for (int i = 1; i < 16; ++i) s += red[i][c];
    void* o = f < b.F ? b.dbg : b.dbu;
    const int at = f < b.F ? f : f - b.F;
    if (o && b.f32) static_cast<float*>(o)[at] = (float)s;
    else if (o) static_cast<T*>(o)[at] = (T)(float)s;
  }
}
template <class T>
__global__ __launch_bounds__(256) void bias_kernel(BiasArgs b) {
  bias_columns<T>(b, blockIdx.x);
}
// A product's partials (n values per split and group) added in order; `blocks` work-groups for each group and, in front
// of them, the bias gradients, which would take a launch of their own (4.4 us, whatever their number)
template <class O, class T>
__global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ part, int64_t n, int parts, int blocks,
                                                      int groups, O* __restrict__ out0, O* __restrict__ out1, BiasArgs b) {
  const int at = (int)blockIdx.x - ((int)gridDim.x - blocks * groups);
  if (at < 0) return bias_columns<T>(b, blockIdx.x);
  const int grp = at >= blocks;
  const int64_t e = (int64_t)(at - grp * blocks) * 256 + threadIdx.x;
  if (e >= n) return;
  part += grp * n + e;
  float s = 0.0f;
  for (int p0 = 0; p0 < parts; p0 += 16) {
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = part[(int64_t)(p0 + k < parts ? p0 + k : p0) * groups * n];
#pragma unroll
    for (int k = 0; k < 16; ++k) s += p0 + k < parts ? v[k] : 0.0f;
  }
  (grp ? out1 : out0)[e] = (O)s;
}

// a plain product (dx, or dWg and dWu as two groups), over splits of k where the plan has them
template <class E, class O, bool NMN, bool MMN>
int run_product(GemmArgs& g, const Plan& p, float* part, const BiasArgs& b, hipStream_t s) {
  if (p.splits == 1) return launch<E, O, NMN, MMN, EPI_OUT, 0>(g, p.tiling, s);
  const int64_t n = g.M * g.N;
  O *o0 = static_cast<O*>(g.out[0]), *o1 = static_cast<O*>(g.out[1]);
  g.splits = p.splits;
  g.kps = p.kps;
  g.out[0] = part;
  g.out[1] = part + n;
  g.o_split = g.groups * n;
  if (int rc = launch<E, float, NMN, MMN, EPI_OUT, 0>(g, p.tiling, s)) return rc;
  const int blocks = (int)cdiv(n, 256), front = b.part ? (int)cdiv(2 * b.F, 16) : 0;
  hipLaunchKernelGGL((combine_kernel<O, typename E::T>), dim3((unsigned)(blocks * g.groups + front)), dim3(256), 0, s, part,
                     n, p.splits, blocks, g.groups, o0, o1, b);
  PCST_LAUNCH_CHECK("gated_linear_bwd");
  return PCST_OK;
}

template <class E>
int bwd_impl(const BwdCall& c, hipStream_t s) {
  typedef typename E::T T;
  constexpr int ES = elem_size<E>();
  const FwdCall& f = c.f;
  GemmArgs g = fwd_args(f);
  g.out[0] = c.dgu;
  g.ldo = 2 * c.fpad;
  g.fpad = c.fpad;
  g.dh = c.dh;
  g.bpart = c.dbg || c.dbu ? c.bpart : nullptr;
  const Plan pg = plan_gated(f.M, f.D, f.F, ES);
  int rc = run_gated<E, T, EPI_BWD>(g, pg, f.act, f.part, s);
  if (rc) return rc;
  BiasArgs bias{g.bpart, (int)f.F, (int)bias_parts(f.M, f.D, f.F, ES, pg), c.bgrad_f32, c.dbg, c.dbu};
  const Plan pw = plan_dw(f.M, f.D, f.F, ES);
  const Plan px = plan_dx(f.M, f.D, f.F, ES);
  const bool with_dx = c.dx && px.splits > 1, with_dw = !with_dx && (c.dwg || c.dwu) && pw.splits > 1;
  if (bias.part && !with_dx && !with_dw) {  // no adding of splits to go with
    hipLaunchKernelGGL(bias_kernel<T>, dim3((unsigned)cdiv(2 * f.F, 16)), dim3(256), 0, s, bias);
    PCST_LAUNCH_CHECK("gated_linear_bwd");
  }
  if (c.dx) {
    GemmArgs d{};
    d.a[0] = static_cast<const char*>(c.dgu);
    d.a[1] = d.a[0] + c.fpad * ES;
    d.b0[0] = static_cast<const char*>(f.wg);
    d.b0[1] = static_cast<const char*>(f.wu);
    d.lda = 2 * c.fpad * ES;
    d.ldb = f.ldw;
    d.M = f.M;
    d.N = (int)f.D;
    d.K = d.kps = f.F;
    d.splits = d.groups = 1;
    d.out[0] = c.dx;
    d.ldo = f.D;
    rc = run_product<E, T, true, false>(d, px, f.part, with_dx ? bias : BiasArgs{}, s);
    if (rc) return rc;
  }
  if (c.dwg || c.dwu) {
    GemmArgs w{};
    w.a[0] = static_cast<const char*>(c.dgu);
    w.b0[0] = static_cast<const char*>(f.x);
    w.lda = 2 * c.fpad * ES;
    w.ldb = f.ldx;
    w.M = f.F;
    w.N = (int)f.D;
    w.K = w.kps = f.M;
    w.splits = 1;
    w.ldo = f.D;
    void* outs[2] = {c.dwg, c.dwu};
    for (int k = 0; k < 2; ++k)
      if (outs[k]) {
        w.a_group[w.groups] = k * c.fpad * ES;
        w.out[w.groups++] = outs[k];
      }
    if (!with_dw) bias = BiasArgs{};
    rc = c.wgrad_f32 ? run_product<E, float, true, true>(w, pw, f.part, bias, s)
                     : run_product<E, T, true, true>(w, pw, f.part, bias, s);
    if (rc) return rc;
  }
  return PCST_OK;
}
#endif  // PCST_GATED_IMPL

}  // namespace gated
}  // namespace pcst
