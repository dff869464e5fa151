// The gated feed-forward block, y = h Wd^T with h = act(g) u, g = x Wg^T, u = x Wu^T, and its backward pass.
//
// Forward, two kernels: one computes both projections of a tile of rows (their weights' rows alternate in its
// second operand, 32 of each, so that a lane holds g and u of the same eight columns), applies the activation
// and the product in registers and writes h and, for the backward pass, g and u; the other is h Wd^T.
//
// Backward: dh = dy Wd is formed tile by tile and never written: its epilogue reads g and u, and writes
// dg = dh u act'(g), du = dh act(g) and h again; then dx = [dg du] [Wg; Wu], d[Wg; Wu] = [dg du]^T x and
// dWd = dy^T h are plain products (product.hip).
//
// bf16 operands: g, u and dh are fp32 sums; h, dg and du are rounded to bf16 once, because they are operands of
// the next bf16 product (2^-8 of each at most, as y itself is rounded).  What is kept of g and u is in blocks of
// 32 columns of a row that share a power of two s: 16 bits (value / s in half precision, 2^-11 of the value; in
// bf16 their rounding was half of the gradients' error, 3.4e-3 of the norm against 2.4e-3), or 8 bits (value / s in
// e4m3, with the smallest s for which |value| <= 448 s).  The backward pass computes with what they stand for.
//
// Up to 64 rows (single tokens of a batch) the time is that of reading the weights once, and a 128-row tile
// would leave most of the chip idle: ffn_rows_kernel gives 16 weight rows to a workgroup, whose waves split k.
#include <algorithm>

#include "product.h"

namespace pnfx {
namespace {

// Phi(g), the normal distribution, and e = exp(-g^2 / 2).  For bf16 operands Phi by formula 7.1.26 of Abramowitz and
// Stegun's Handbook of Mathematical Functions for erf of |g| / sqrt 2, which uses the same e: within 1.5e-7 of erf in exact
// arithmetic, Phi within 3e-7 with the roundings of fp32, and of its lower tail a share of 2e-3 (g = -5) to 1e-2 (-8); h,
// dg and du are rounded to bf16, 4e-3.  For fp32 operands it is the library's erfc, which keeps the tail's digits (4096 x
// 256 x 1024 rows: training 226 -> 229 us, inference 67 -> 69; 16384 x 64 x 512: 221 -> 230, 54 -> 59).
template <typename T>
__device__ __forceinline__ float phi(float g, float& e) {
  if constexpr (sizeof(T) == 4) {
    e = __expf(-0.5f * g * g);
    return 0.5f * erfcf(-0.70710678118654752f * g);
  }
  const float x = fabsf(g) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, x, 1.f));
  e = __expf(-x * x);
  float q = __builtin_fmaf(1.061405429f, t, -1.453152027f);
  q = __builtin_fmaf(q, t, 1.421413741f);
  q = __builtin_fmaf(q, t, -0.284496736f);
  q = __builtin_fmaf(q, t, 0.254829592f);
  q *= 0.5f * t * e;
  return g >= 0.f ? 1.f - q : q;
}
template <typename T, int ACT>
__device__ __forceinline__ float act_of(float g) {
  if constexpr (ACT == PNFX_ACT_SILU) return g * __builtin_amdgcn_rcpf(1.f + __expf(-g));
  float e;
  return g * phi<T>(g, e);
}
// act(g) and act'(g)
template <typename T, int ACT>
__device__ __forceinline__ void act_both(float g, float& a, float& d) {
  if constexpr (ACT == PNFX_ACT_SILU) {
    const float p = __builtin_amdgcn_rcpf(1.f + __expf(-g));
    a = g * p;
    d = p * (1.f + g * (1.f - p));
  } else {
    float e;
    const float p = phi<T>(g, e);
    a = g * p;
    d = p + g * 0.39894228040143268f * e;
  }
}

// -------------------------------------------------------------------- blocks of 32
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
// The largest finite |v| of the lane's eight values and the other three lanes' of the row's 32.
__device__ __forceinline__ float block_top(const float* v) {
  float t = 0.f;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const float a = fabsf(v[r]);
    t = fmaxf(t, a < INFINITY ? a : 0.f);
  }
  t = fmaxf(t, __shfl_xor(t, 16, 64));
  return fmaxf(t, __shfl_xor(t, 32, 64));
}
// Exponent of the power of two that brings a block into half precision's range: values below 2^15.
__device__ __forceinline__ int half_exp(float top) { return max((int)(__float_as_uint(top) >> 23) - 127 - 14, -126); }
// Exponent of the smallest power of two s with top <= 448 s (448 = 1.75 2^8), at least -126.
__device__ __forceinline__ int scale_exp(float top) {
  const unsigned b = __float_as_uint(top);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffff) > 0x600000);
  return max(e, -126);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
// Four values over s as e4m3.
__device__ __forceinline__ uint32_t pack_e4m3(const float* v, float inv) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, w, true);
}
__device__ __forceinline__ void unpack_e4m3(uint32_t w, float s, float* v) {
  v[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0) * s;
  v[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * s;
  v[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * s;
  v[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * s;
}

// Fp: F rounded up to a multiple of 8, the columns of h, of either half of g | u and of either half of dg | du;
// those past F are zero.
struct GluArgs {
  const void* x;    // [T][ldx], or dy
  const void* wg;   // [F][ldw], or Wd [Do][ldw]
  const void* wu;
  void* h;          // [T][Fp]
  void* gu;         // [T][2 Fp]: fp32, or half precision or bytes in blocks; null: not kept
  uint8_t* scales;  // [T][2 nb]: exponent + 127 of each block's power of two
  void* dgu;        // [T][2 Fp]
  int64_t ldx, ldw, K;
  int T, F, Fp, nb, tm, tn;
  int keep;
};

template <typename T, int ACT, class C>
__global__ __launch_bounds__(threads_of<C>, 2) void glu_fwd_kernel(GluArgs a) {
  typedef Product<T, ROW, PAIR, C> P;
  extern __shared__ __align__(16) char sm[];
  int tm, tn;
  tile_of(blockIdx.x, a.tm, a.tn, tm, tn);
  const int m0 = tm * C::TM, f0 = tn * (C::TN / 2);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  typename P::StageA sa;
  typename P::StageB sb;
  sa.init(static_cast<const T*>(a.x) + m0 * a.ldx, a.ldx, a.T - m0, a.K, threadIdx.x);
  sb.init(static_cast<const T*>(a.wg) + f0 * a.ldw, a.ldw, a.F - f0, a.K, threadIdx.x,
          static_cast<const T*>(a.wu) + f0 * a.ldw);
  f32x4 acc[P::MI][P::NJ] = {};
  P::run(sa, sb, (int)((a.K + k_step<T> - 1) / k_step<T>), reinterpret_cast<T*>(sm), wave, lane, acc);
  const int wm = wave / C::WN * P::MI, wn = wave % C::WN * P::NJ, ag = lane >> 4;
  // columns past F are of zero weights: zero for any x, an infinite one too
  if (f0 + C::TN / 2 > a.F) {
#pragma unroll
    for (int j = 0; j < P::NJ; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (f0 + 32 * ((wn + j) / 4) + 8 * ag + 4 * (j & 1) + r >= a.F) {
#pragma unroll
          for (int i = 0; i < P::MI; ++i) acc[i][j][r] = 0.f;
        }
  }
#pragma unroll
  for (int i = 0; i < P::MI; ++i) {
    const int m = m0 + stage_row<ROW>(wm + i, lane & 15);
#pragma unroll
    for (int s = 0; s < P::NJ / 4; ++s) {
      const int fb = f0 + 32 * (wn / 4 + s), f = fb + 8 * ag;  // the 32 columns' first, the lane's first of 8
      float g[8], u[8], h[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        g[r] = acc[i][4 * s + (r >> 2)][r & 3];
        u[r] = acc[i][4 * s + 2 + (r >> 2)][r & 3];
        h[r] = act_of<T, ACT>(g[r]) * u[r];
      }
      const bool in = m < a.T && f < a.Fp;
      if (in) store8(static_cast<T*>(a.h) + (int64_t)m * a.Fp + f, h);
      if (a.keep == PNFX_KEEP_NONE) continue;
      const int64_t at = (int64_t)m * 2 * a.Fp + f;
      if constexpr (sizeof(T) == 4) {
        if (in) {
          store8(static_cast<float*>(a.gu) + at, g);
          store8(static_cast<float*>(a.gu) + at + a.Fp, u);
        }
      } else {
        // columns past F change no maximum
        const float tg = block_top(g), tu = block_top(u);
        const bool half = a.keep == PNFX_KEEP_FULL;
        const int eg = half ? half_exp(tg) : scale_exp(tg), eu = half ? half_exp(tu) : scale_exp(tu);
        const float ig = pow2(-eg), iu = pow2(-eu);
        if (!in) continue;
        if (half) {
          f16x8 hg, hu;
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            hg[r] = (_Float16)(g[r] * ig);
            hu[r] = (_Float16)(u[r] * iu);
          }
          _Float16* gu = static_cast<_Float16*>(a.gu) + at;
          *reinterpret_cast<f16x8*>(gu) = hg;
          *reinterpret_cast<f16x8*>(gu + a.Fp) = hu;
        } else {
          uint8_t* gu = static_cast<uint8_t*>(a.gu) + at;
          *reinterpret_cast<uint2*>(gu) = uint2{pack_e4m3(g, ig), pack_e4m3(g + 4, ig)};
          *reinterpret_cast<uint2*>(gu + a.Fp) = uint2{pack_e4m3(u, iu), pack_e4m3(u + 4, iu)};
        }
        if (ag == 0) {
          uint8_t* sc = a.scales + (int64_t)m * 2 * a.nb + fb / 32;
          sc[0] = (uint8_t)(eg + 127);
          sc[a.nb] = (uint8_t)(eu + 127);
        }
      }
    }
  }
}

// Eight columns of g and u as they were kept, from memory and as fp32.
template <typename T>
struct KeptPart;
template <>
struct KeptPart<float> {
  f32x4 g[2], u[2];
  __device__ __forceinline__ void load(const GluArgs& a, int m, int f, int) {
    const float* p = static_cast<const float*>(a.gu) + (int64_t)m * 2 * a.Fp + f;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      g[r] = *reinterpret_cast<const f32x4*>(p + 4 * r);
      u[r] = *reinterpret_cast<const f32x4*>(p + a.Fp + 4 * r);
    }
  }
  __device__ __forceinline__ void get(int, float* vg, float* vu) const {
#pragma unroll
    for (int r = 0; r < 8; ++r) vg[r] = g[r >> 2][r & 3], vu[r] = u[r >> 2][r & 3];
  }
};
template <>
struct KeptPart<bf16> {
  uint4 g, u;  // e4m3: the first half of each
  uint8_t sg, su;
  __device__ __forceinline__ void load(const GluArgs& a, int m, int f, int block) {
    const int64_t at = (int64_t)m * 2 * a.Fp + f;
    if (a.keep == PNFX_KEEP_FULL) {
      const _Float16* p = static_cast<const _Float16*>(a.gu) + at;
      g = *reinterpret_cast<const uint4*>(p);
      u = *reinterpret_cast<const uint4*>(p + a.Fp);
    } else {
      const uint8_t* p = static_cast<const uint8_t*>(a.gu) + at;
      const uint2 g2 = *reinterpret_cast<const uint2*>(p), u2 = *reinterpret_cast<const uint2*>(p + a.Fp);
      g.x = g2.x, g.y = g2.y, u.x = u2.x, u.y = u2.y;
    }
    const uint8_t* sc = a.scales + (int64_t)m * 2 * a.nb + block;
    sg = sc[0];
    su = sc[a.nb];
  }
  __device__ __forceinline__ void get(int keep, float* vg, float* vu) const {
    const float fg = pow2((int)sg - 127), fu = pow2((int)su - 127);
    if (keep == PNFX_KEEP_FULL) {
      const f16x8 hg = __builtin_bit_cast(f16x8, g), hu = __builtin_bit_cast(f16x8, u);
#pragma unroll
      for (int r = 0; r < 8; ++r) vg[r] = (float)hg[r] * fg, vu[r] = (float)hu[r] * fu;
    } else {
      unpack_e4m3(g.x, fg, vg);
      unpack_e4m3(g.y, fg, vg + 4);
      unpack_e4m3(u.x, fu, vu);
      unpack_e4m3(u.y, fu, vu + 4);
    }
  }
};

template <typename T, int ACT, class C>
__global__ __launch_bounds__(threads_of<C>, 2) void glu_bwd_kernel(GluArgs a) {
  typedef Product<T, ROW, COL, C> P;
  extern __shared__ __align__(16) char sm[];
  int tm, tn;
  tile_of(blockIdx.x, a.tm, a.tn, tm, tn);
  const int m0 = tm * C::TM, n0 = tn * C::TN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  typename P::StageA sa;
  typename P::StageB sb;
  sa.init(static_cast<const T*>(a.x) + m0 * a.ldx, a.ldx, a.T - m0, a.K, threadIdx.x);
  sb.init(static_cast<const T*>(a.wg) + n0, a.ldw, a.F - n0, a.K, threadIdx.x);
  f32x4 acc[P::MI][P::NJ] = {};
  P::run(sa, sb, (int)((a.K + k_step<T> - 1) / k_step<T>), reinterpret_cast<T*>(sm), wave, lane, acc);
  const int wm = wave / C::WN * P::MI, wn = wave % C::WN * P::NJ;
  // g and u of one row block are read while the block before is worked on
  typedef KeptPart<T> Part;
  constexpr int NP = P::NJ / 2;  // pairs of blocks: eight columns of a lane, 32 of a wave
  Part part[2][NP];
  const auto fetch = [&](int i) {
    const int m = min(m0 + stage_row<ROW>(wm + i, lane & 15), a.T - 1);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int f = n0 + pair_col<COL>(wn + 2 * p, lane);
      part[i & 1][p].load(a, m, min(f, a.Fp - 8), min((n0 + 16 * (wn + 2 * p)) / 32, a.nb - 1));
    }
  };
  fetch(0);
#pragma unroll
  for (int i = 0; i < P::MI; ++i) {
    if (i + 1 < P::MI) fetch(i + 1);
    __builtin_amdgcn_sched_barrier(0);
    const int m = m0 + stage_row<ROW>(wm + i, lane & 15);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int f = n0 + pair_col<COL>(wn + 2 * p, lane);
      float dh[8], g[8], u[8], dg[8], du[8], h[8];
      pair8<COL>(acc[i][2 * p], acc[i][2 * p + 1], dh);
      part[i & 1][p].get(a.keep, g, u);
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        float s, d;
        act_both<T, ACT>(g[r], s, d);
        // columns between F and Fp are of zero weights: zero for any dy, an infinite one too
        const float v = f + r < a.F ? dh[r] : 0.f;
        dg[r] = v * u[r] * d;
        du[r] = v * s;
        h[r] = s * u[r];
      }
      if (m >= a.T || f >= a.Fp) continue;
      T* o = static_cast<T*>(a.dgu) + (int64_t)m * 2 * a.Fp + f;
      store8(o, dg);
      store8(o + a.Fp, du);
      store8(static_cast<T*>(a.h) + (int64_t)m * a.Fp + f, h);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// ------------------------------------------------------------------------ few rows
// Up to here ffn_rows_kernel takes them (us of a call, bf16, this kernel / the tiles: 17 rows, D = 1024, F = 4096 10.9 /
// 21.8; 64 rows 16.3 / 25.5; 64 rows, D = 2048, F = 8192 33.5 / 40.9; D = 4096, F = 11008 73 / 91; beyond, its four
// blocks of 16 rows would not do).
constexpr int kFewRows = 64;

struct RowsArgs {
  const void* x;   // [T][ldx]
  const void* w;   // [N][ldw]
  const void* w2;  // PAIRED: the up projection
  void* y;         // [T][ldy]
  int64_t ldx, ldw, ldy;
  int T, N, K, cols;  // cols: columns of y to write, those past N as zeros
};

// y[t][n] = sum_k x[t][k] w[n][k], or with PAIRED act(that) times the same with w2: 16 n per workgroup, MB blocks of
// 16 rows t; wave w takes the 128-byte pieces of k number w, w + W, ...  Each wave brings its pieces of the weights
// and of x to LDS of its own, S pieces ahead and without a barrier, eight lanes to a row: read straight into
// registers in the products' layout, 16 rows side by side, every lane is a cache access of its own (39 for each load
// of 1 KB, and the address unit busy throughout).  Zeros past N, T and K.
template <bool PAIRED, int MB>
struct FewRows {
  static constexpr int W = PAIRED ? 4 : 8;                      // waves
  static constexpr int PARTS = (PAIRED ? 2 : 1) + MB;           // 16-row parts of a piece, 2 KB each
  static constexpr int S = PARTS <= (PAIRED ? 3 : 2) ? 4 : PARTS <= (PAIRED ? 4 : 3) ? 3 : 2;  // pieces on their way
  static constexpr int LDS = W * S * PARTS * 2048;
  static_assert(LDS <= 160 * 1024, "a CU's LDS");
};
template <typename T, int ACT, bool PAIRED, int MB>
__global__ __launch_bounds__((64 * FewRows<PAIRED, MB>::W), 2) void ffn_rows_kernel(RowsArgs a) {
  typedef typename Elem<T>::Frag F;
  typedef FewRows<PAIRED, MB> R;
  constexpr int ES = (int)sizeof(T), W = R::W, S = R::S, PARTS = R::PARTS, NM = PAIRED ? 2 : 1;
  constexpr int PART = 2048 / ES;  // elements
  extern __shared__ __align__(16) char sm[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r16 = lane & 15, g = lane >> 4, n0 = blockIdx.x * 16;
  const unsigned rows = (unsigned)min(a.N - n0, 16), kb = (unsigned)a.K * ES;
  const unsigned ldw = (unsigned)(a.ldw * ES), ldx = (unsigned)(a.ldx * ES);
  const u32x4 dw = buffer_of(static_cast<const T*>(a.w) + n0 * a.ldw, (rows - 1) * ldw + kb);
  const u32x4 du = PAIRED ? buffer_of(static_cast<const T*>(a.w2) + n0 * a.ldw, (rows - 1) * ldw + kb) : dw;
  const u32x4 dx = buffer_of(a.x, (unsigned)(a.T - 1) * ldx + kb);
  // a load fills eight slots: lane l the chunk that belongs at position l % 8 of slot l / 8 (and slot + 8)
  const int slot = lane >> 3, c0 = (lane & 7) ^ stage_swz<T, ROW>(slot), c1 = (lane & 7) ^ stage_swz<T, ROW>(slot + 8);
  T* const ring = reinterpret_cast<T*>(sm) + wave * (S * PARTS * PART);
  const unsigned at = __builtin_amdgcn_readfirstlane(lds_addr(ring));
  const auto fetch = [&](int stage, unsigned piece) {
    const unsigned k0 = piece * 128 + 16 * c0, k1 = piece * 128 + 16 * c1;
    const auto part = [&](u32x4 d, unsigned ld, int first, int p) {
      const unsigned to = at + (stage * PARTS + p) * 2048;
      lds_dma16(d, k0 < kb ? (first + slot) * ld + k0 : 0x80000000u, to);
      lds_dma16(d, k1 < kb ? (first + slot + 8) * ld + k1 : 0x80000000u, to + 1024);
    };
    part(dw, ldw, 0, 0);
    if constexpr (PAIRED) part(du, ldw, 0, 1);
#pragma unroll
    for (int b = 0; b < MB; ++b) part(dx, ldx, 16 * b, NM + b);
  };
  const T* frag[2];
#pragma unroll
  for (int hf = 0; hf < 2; ++hf)
    frag[hf] = ring + r16 * (128 / ES) + per16<T> * ((g + 4 * hf) ^ stage_swz<T, ROW>(r16));
  f32x4 acc[NM][MB] = {};
  const unsigned pieces = (kb + 127) / 128;
#pragma unroll
  for (int s = 0; s < S; ++s) fetch(s, wave + s * W);
  int stage = 0;
  for (unsigned p = wave; p < pieces; p += W) {
    wait_vm_lgkm<(S - 1) * PARTS * 2>();
    F f[2][PARTS];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int q = 0; q < PARTS; ++q)
        f[hf][q] = *reinterpret_cast<const F*>(frag[hf] + (stage * PARTS + q) * PART);
    wait_vm_lgkm<63>();
    __builtin_amdgcn_sched_barrier(0);
    fetch(stage, p + S * W);  // past the last piece: zeros, so that the count of loads is the same
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int m = 0; m < NM; ++m) acc[m][b] = mma(f[hf][m], f[hf][NM + b], acc[m][b]);
    stage = stage + 1 == S ? 0 : stage + 1;
  }
  wait_vm_lgkm<0>();
  __syncthreads();
  f32x4(*const part)[NM * MB][64] = reinterpret_cast<f32x4(*)[NM * MB][64]>(sm);
  static_assert((W - 1) * NM * MB * 1024 <= R::LDS, "");
  // the waves' sums, added in wave order
  if (wave) {
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
      for (int b = 0; b < MB; ++b) part[wave - 1][m * MB + b][lane] = acc[m][b];
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int v = 0; v < W - 1; ++v)
#pragma unroll
    for (int m = 0; m < NM; ++m)
#pragma unroll
      for (int b = 0; b < MB; ++b) acc[m][b] += part[v][m * MB + b][lane];
#pragma unroll
  for (int b = 0; b < MB; ++b) {
    const int t = 16 * b + r16;
    if (t >= a.T) continue;
    T* y = static_cast<T*>(a.y) + t * a.ldy;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = n0 + 4 * g + r;
      const float v = PAIRED ? act_of<T, ACT>(acc[0][b][r]) * acc[NM - 1][b][r] : acc[0][b][r];
      if (n < a.cols) y[n] = from_f32<T>(n < a.N ? v : 0.f);  // (zero weights past N, but x may be infinite)
    }
  }
}

template <typename T, int ACT, bool PAIRED, int MB>
int rows_launch(const RowsArgs& a, hipStream_t st) {
  typedef FewRows<PAIRED, MB> R;
  return launch<ffn_rows_kernel<T, ACT, PAIRED, MB>>(ceil_div(a.cols, 16), 64 * R::W, R::LDS, a, st, "ffn rows");
}
template <typename T, int ACT, bool PAIRED>
int rows_any(const RowsArgs& a, hipStream_t st) {
  if (a.T <= 16) return rows_launch<T, ACT, PAIRED, 1>(a, st);
  if (a.T <= 32) return rows_launch<T, ACT, PAIRED, 2>(a, st);
  if (a.T <= 48) return rows_launch<T, ACT, PAIRED, 3>(a, st);
  return rows_launch<T, ACT, PAIRED, 4>(a, st);
}

// ------------------------------------------------------------------------ host side
struct Sizes {
  int64_t T, D, F, Do, Dp, Fp, Dop, nb;
  int es, dtype;
};
Sizes sizes_of(int64_t T, int64_t D, int64_t F, int64_t Do, int dtype) {
  Sizes z;
  z.T = T, z.D = D, z.F = F, z.Do = Do;
  z.Dp = round_up(D, 8), z.Fp = round_up(F, 8), z.Dop = round_up(Do, 8);
  z.nb = ceil_div(F, 32);
  z.es = dtype == PNFX_F32 ? 4 : 2;
  z.dtype = dtype;
  return z;
}

// Workspace handed out in pieces of 256 bytes; null: only counted.
struct Arena {
  char* p;
  int64_t used;
  void* take(int64_t bytes) {
    char* r = p ? p + used : nullptr;
    used += round_up(bytes, 256);
    return r;
  }
};

// An operand as the kernels take it: in place, or a padded copy.
struct In {
  const void* p;
  int64_t ld;
};
bool in_place(const void* p, int64_t ld, int64_t cols, const Sizes& z) {
  return cols % 8 == 0 && operand_ok(p, ld, z.es);
}

int check_sizes(const char* what, int64_t T, int64_t D, int64_t F, int64_t Do, int act, int dtype) {
  PNFX_REQUIRE(dtype == PNFX_F32 || dtype == PNFX_BF16, "%s: unsupported dtype %d", what, dtype);
  PNFX_REQUIRE(act == PNFX_ACT_SILU || act == PNFX_ACT_GELU, "%s: unknown activation %d", what, act);
  PNFX_REQUIRE(T >= 1 && D >= 1 && F >= 1 && Do >= 1 && T < (1 << 29) && D <= (1 << 18) && F <= (1 << 18) &&
                   Do <= (1 << 18),
               "%s: bad shape T=%lld D=%lld F=%lld Do=%lld", what, (long long)T, (long long)D, (long long)F,
               (long long)Do);
  return PNFX_OK;
}

// The padded copies that a call makes of what it cannot take in place.
struct Operands {
  PadItem pads[4];
  int n = 0;
  In take(Arena& ar, const void* p, int64_t ld, int64_t rows, int64_t cols, const Sizes& z) {
    if (in_place(p, ld, cols, z)) return In{p, ld};
    const int64_t cp = round_up(cols, 8);
    void* d = ar.take(rows * cp * z.es);
    pads[n++] = PadItem{p, d, ld, rows, cols, rows, cp, 1};
    return In{d, cp};
  }
  // both halves of w_in, Fp rows apart
  In take_in(Arena& ar, const void* p, int64_t ld, const Sizes& z) {
    if (z.F == z.Fp && in_place(p, ld, z.D, z)) return In{p, ld};
    void* d = ar.take(2 * z.Fp * z.Dp * z.es);
    pads[n++] = PadItem{p, d, ld, z.F, z.D, z.Fp, z.Dp, 2};
    return In{d, z.Dp};
  }
};

template <typename T, int ACT>
int glu_fwd(GluArgs& a, bool big, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (big) {
      a.tm = (int)ceil_div(a.T, Big::TM), a.tn = (int)ceil_div(a.Fp, Big::TN / 2);
      return launch<glu_fwd_kernel<T, ACT, Big>>((int64_t)a.tm * a.tn, threads_of<Big>, lds_of<Big>, a, st, "glu_fwd");
    }
  }
  a.tm = (int)ceil_div(a.T, Mid::TM), a.tn = (int)ceil_div(a.Fp, Mid::TN / 2);
  return launch<glu_fwd_kernel<T, ACT, Mid>>((int64_t)a.tm * a.tn, threads_of<Mid>, lds_of<Mid>, a, st, "glu_fwd");
}
template <typename T, int ACT>
int glu_bwd(GluArgs& a, bool big, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (big) {
      a.tm = (int)ceil_div(a.T, Big::TM), a.tn = (int)ceil_div(a.Fp, Big::TN);
      return launch<glu_bwd_kernel<T, ACT, Big>>((int64_t)a.tm * a.tn, threads_of<Big>, lds_of<Big>, a, st, "glu_bwd");
    }
  }
  a.tm = (int)ceil_div(a.T, Mid::TM), a.tn = (int)ceil_div(a.Fp, Mid::TN);
  return launch<glu_bwd_kernel<T, ACT, Mid>>((int64_t)a.tm * a.tn, threads_of<Mid>, lds_of<Mid>, a, st, "glu_bwd");
}

struct FwdArgs {
  const void *x, *w_in, *w_down;
  int64_t x_rs, win_rs, wd_rs;
  void *y, *gu;
  uint8_t* scales;
  int act, keep;
};

// Workspace of the forward pass, with or without padded copies of its operands.
bool few_rows(const Sizes& z, int keep) { return z.T <= kFewRows && keep == PNFX_KEEP_NONE; }
int64_t fwd_bytes(const Sizes& z, int keep, bool copies) {
  Arena ar{nullptr, 0};
  if (copies) {
    ar.take(z.T * z.Dp * z.es);
    ar.take(2 * z.Fp * z.Dp * z.es);
    ar.take(z.Do * z.Fp * z.es);
  }
  ar.take(z.T * z.Fp * z.es);
  if (!few_rows(z, keep)) ar.take(product_workspace(cut_of(z.T, z.Do, z.Fp, z.dtype, true), z.T, z.Do));
  return ar.used;
}

template <typename T, int ACT>
int ffn_fwd(const FwdArgs& f, const Sizes& z, void* ws, hipStream_t st) {
  Arena ar{static_cast<char*>(ws), 0};
  Operands ops;
  const In x = ops.take(ar, f.x, f.x_rs, z.T, z.D, z);
  const In win = ops.take_in(ar, f.w_in, f.win_rs, z);
  const In wd = ops.take(ar, f.w_down, f.wd_rs, z.Do, z.F, z);
  void* h = ar.take(z.T * z.Fp * z.es);
  PNFX_TRY(pad(ops.pads, ops.n, z.dtype, st));
  const T* wg = static_cast<const T*>(win.p);
  const T* wu = wg + z.Fp * win.ld;
  if (few_rows(z, f.keep)) {
    RowsArgs r{x.p, wg, wu, h, x.ld, win.ld, z.Fp, (int)z.T, (int)z.F, (int)z.Dp, (int)z.Fp};
    PNFX_TRY((rows_any<T, ACT, true>(r, st)));
    RowsArgs d{h, wd.p, nullptr, f.y, z.Fp, wd.ld, z.Do, (int)z.T, (int)z.Do, (int)z.Fp, (int)z.Do};
    return rows_any<T, ACT, false>(d, st);
  }
  GluArgs a = {};
  a.x = x.p, a.wg = wg, a.wu = wu, a.h = h, a.gu = f.gu, a.scales = f.scales;
  a.ldx = x.ld, a.ldw = win.ld, a.K = z.Dp;
  a.T = (int)z.T, a.F = (int)z.F, a.Fp = (int)z.Fp, a.nb = (int)z.nb, a.keep = f.keep;
  PNFX_TRY((glu_fwd<T, ACT>(a, cut_of(z.T, 2 * z.Fp, z.Dp, z.dtype, false).big(), st)));
  const Cut cut = cut_of(z.T, z.Do, z.Fp, z.dtype, true);
  ProductArgs p = {};
  p.a = h, p.b = wd.p, p.c = f.y, p.lda = z.Fp, p.ldb = wd.ld, p.ldc = z.Do;
  p.M = z.T, p.N = z.Do, p.K = z.Fp;
  const Job job{ROW, ROW, p, cut, ar.take(product_workspace(cut, z.T, z.Do))};
  return products(&job, 1, z.dtype, st);
}

// dx, dw_in, dw_down
void bwd_cuts(const Sizes& z, Shape* s, Cut* cuts) {
  s[0] = Shape{z.T, z.D, 2 * z.Fp, false};
  s[1] = Shape{z.Fp + z.F, z.D, z.T, false};
  s[2] = Shape{z.Do, z.F, z.T, false};
  cut_group(s, 3, z.dtype, true, cuts);
}
int64_t bwd_bytes(const Sizes& z, bool copies) {
  Arena ar{nullptr, 0};
  if (copies) {
    ar.take(z.T * z.Dop * z.es);
    ar.take(z.T * z.Dp * z.es);
    ar.take(2 * z.Fp * z.Dp * z.es);
    ar.take(z.Do * z.Fp * z.es);
  }
  ar.take(z.T * 2 * z.Fp * z.es);
  ar.take(z.T * z.Fp * z.es);
  Shape s[3];
  Cut cuts[3];
  bwd_cuts(z, s, cuts);
  for (int i = 0; i < 3; ++i) ar.take(product_workspace(cuts[i], s[i].M, s[i].N));
  return ar.used;
}

struct BwdArgs {
  const void *dy, *x, *w_in, *w_down, *gu;
  const uint8_t* scales;
  int64_t dy_rs, x_rs, win_rs, wd_rs;
  void *dx, *dw_in, *dw_down;
  int act, keep;
};

template <typename T, int ACT>
int ffn_bwd(const BwdArgs& f, const Sizes& z, void* ws, hipStream_t st) {
  Arena ar{static_cast<char*>(ws), 0};
  Operands ops;
  const In dy = ops.take(ar, f.dy, f.dy_rs, z.T, z.Do, z);
  const In x = ops.take(ar, f.x, f.x_rs, z.T, z.D, z);
  const In win = ops.take_in(ar, f.w_in, f.win_rs, z);
  const In wd = ops.take(ar, f.w_down, f.wd_rs, z.Do, z.F, z);
  void* dgu = ar.take(z.T * 2 * z.Fp * z.es);
  void* h = ar.take(z.T * z.Fp * z.es);
  Shape s[3];
  Cut cuts[3];
  bwd_cuts(z, s, cuts);
  PNFX_TRY(pad(ops.pads, ops.n, z.dtype, st));
  GluArgs a = {};
  a.x = dy.p, a.wg = wd.p, a.h = h, a.gu = const_cast<void*>(f.gu), a.scales = const_cast<uint8_t*>(f.scales);
  a.dgu = dgu, a.ldx = dy.ld, a.ldw = wd.ld, a.K = z.Do;
  a.T = (int)z.T, a.F = (int)z.F, a.Fp = (int)z.Fp, a.nb = (int)z.nb, a.keep = f.keep;
  PNFX_TRY((glu_bwd<T, ACT>(a, cut_of(z.T, z.Fp, z.Do, z.dtype, false).big(), st)));
  Job jobs[3];
  int n = 0;
  const auto job = [&](int i, int ka, const void* pa, int64_t lda, const void* pb, int64_t ldb, void* c, int64_t ldc) {
    void* sums = ar.take(product_workspace(cuts[i], s[i].M, s[i].N));
    if (!c) return;
    ProductArgs p = {};
    p.a = pa, p.b = pb, p.c = c, p.lda = lda, p.ldb = ldb, p.ldc = ldc;
    p.M = s[i].M, p.N = s[i].N, p.K = s[i].K;
    // dw_in: the columns of dg behind F are no rows of it (those of du behind F are left out as the last ones)
    if (i == 1) p.gap_at = z.F, p.gap = z.Fp - z.F;
    jobs[n++] = Job{ka, COL, p, cuts[i], sums};
  };
  job(0, ROW, dgu, 2 * z.Fp, win.p, win.ld, f.dx, z.D);
  job(1, COL, dgu, 2 * z.Fp, x.p, x.ld, f.dw_in, z.D);
  job(2, COL, dy.p, dy.ld, h, z.Fp, f.dw_down, z.F);
  return n ? products(jobs, n, z.dtype, st) : PNFX_OK;
}

}  // namespace
}  // namespace pnfx

extern "C" int64_t pnfx_ffn_fwd_workspace_size(int64_t T, int64_t D, int64_t F, int64_t Do, int keep, int copies,
                                               int dtype) {
  using namespace pnfx;
  if (check_sizes("ffn", T, D, F, Do, PNFX_ACT_SILU, dtype) != PNFX_OK) return 0;
  return fwd_bytes(sizes_of(T, D, F, Do, dtype), keep, copies);
}

extern "C" int pnfx_ffn_fwd(const void* x, int64_t x_rs, const void* w_in, int64_t win_rs, const void* w_down,
                            int64_t wd_rs, void* y, void* gu, uint8_t* scales, int64_t T, int64_t D, int64_t F,
                            int64_t Do, int act, int keep, int dtype, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  using namespace pnfx;
  PNFX_REQUIRE(x && w_in && w_down && y, "ffn_fwd: null pointer");
  PNFX_TRY(check_sizes("ffn_fwd", T, D, F, Do, act, dtype));
  PNFX_REQUIRE(keep == PNFX_KEEP_NONE || keep == PNFX_KEEP_FULL || (keep == PNFX_KEEP_E4M3 && dtype == PNFX_BF16),
               "ffn_fwd: keep %d of dtype %d", keep, dtype);
  PNFX_REQUIRE(keep == PNFX_KEEP_NONE || (gu && (dtype == PNFX_F32 || scales)), "ffn_fwd: nowhere to keep g and u");
  PNFX_REQUIRE(x_rs >= D && win_rs >= D && wd_rs >= F, "ffn_fwd: row strides %lld, %lld, %lld", (long long)x_rs,
               (long long)win_rs, (long long)wd_rs);
  const Sizes z = sizes_of(T, D, F, Do, dtype);
  PNFX_REQUIRE(((reinterpret_cast<uintptr_t>(gu) | reinterpret_cast<uintptr_t>(workspace) |
                 reinterpret_cast<uintptr_t>(y)) & 15) == 0,
               "ffn_fwd: results and workspace must be 16-byte aligned");
  const bool copies = !(in_place(x, x_rs, D, z) && z.F == z.Fp && in_place(w_in, win_rs, D, z) &&
                        in_place(w_down, wd_rs, F, z));
  const int64_t need = fwd_bytes(z, keep, copies);
  PNFX_REQUIRE(workspace && workspace_bytes >= need, "ffn_fwd: workspace needs %lld bytes", (long long)need);
  const FwdArgs f{x, w_in, w_down, x_rs, win_rs, wd_rs, y, gu, scales, act, keep};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == PNFX_F32)
    return act == PNFX_ACT_SILU ? ffn_fwd<float, PNFX_ACT_SILU>(f, z, workspace, st)
                                : ffn_fwd<float, PNFX_ACT_GELU>(f, z, workspace, st);
  return act == PNFX_ACT_SILU ? ffn_fwd<bf16, PNFX_ACT_SILU>(f, z, workspace, st)
                              : ffn_fwd<bf16, PNFX_ACT_GELU>(f, z, workspace, st);
}

extern "C" int64_t pnfx_ffn_bwd_workspace_size(int64_t T, int64_t D, int64_t F, int64_t Do, int copies, int dtype) {
  using namespace pnfx;
  if (check_sizes("ffn", T, D, F, Do, PNFX_ACT_SILU, dtype) != PNFX_OK) return 0;
  return bwd_bytes(sizes_of(T, D, F, Do, dtype), copies);
}

extern "C" int pnfx_ffn_bwd(const void* dy, int64_t dy_rs, const void* x, int64_t x_rs, const void* w_in,
                            int64_t win_rs, const void* w_down, int64_t wd_rs, const void* gu, const uint8_t* scales,
                            void* dx, void* dw_in, void* dw_down, int64_t T, int64_t D, int64_t F, int64_t Do, int act,
                            int keep, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace pnfx;
  PNFX_REQUIRE(dy && x && w_in && w_down && gu, "ffn_bwd: null pointer");
  PNFX_TRY(check_sizes("ffn_bwd", T, D, F, Do, act, dtype));
  PNFX_REQUIRE(dtype == PNFX_F32 ? keep == PNFX_KEEP_FULL
                                 : (keep == PNFX_KEEP_FULL || keep == PNFX_KEEP_E4M3) && scales,
               "ffn_bwd: keep %d of dtype %d", keep, dtype);
  PNFX_REQUIRE(dy_rs >= Do && x_rs >= D && win_rs >= D && wd_rs >= F, "ffn_bwd: row strides %lld, %lld, %lld, %lld",
               (long long)dy_rs, (long long)x_rs, (long long)win_rs, (long long)wd_rs);
  const Sizes z = sizes_of(T, D, F, Do, dtype);
  PNFX_REQUIRE(((reinterpret_cast<uintptr_t>(gu) | reinterpret_cast<uintptr_t>(workspace) |
                 reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(dw_in) |
                 reinterpret_cast<uintptr_t>(dw_down)) & 15) == 0,
               "ffn_bwd: results, g and u and the workspace must be 16-byte aligned");
  const bool copies = !(in_place(dy, dy_rs, Do, z) && in_place(x, x_rs, D, z) && z.F == z.Fp &&
                        in_place(w_in, win_rs, D, z) && in_place(w_down, wd_rs, F, z));
  const int64_t need = bwd_bytes(z, copies);
  PNFX_REQUIRE(workspace && workspace_bytes >= need, "ffn_bwd: workspace needs %lld bytes", (long long)need);
  const BwdArgs f{dy, x, w_in, w_down, gu, scales, dy_rs, x_rs, win_rs, wd_rs, dx, dw_in, dw_down, act, keep};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == PNFX_F32)
    return act == PNFX_ACT_SILU ? ffn_bwd<float, PNFX_ACT_SILU>(f, z, workspace, st)
                                : ffn_bwd<float, PNFX_ACT_GELU>(f, z, workspace, st);
  return act == PNFX_ACT_SILU ? ffn_bwd<bf16, PNFX_ACT_SILU>(f, z, workspace, st)
                              : ffn_bwd<bf16, PNFX_ACT_GELU>(f, z, workspace, st);
}
