// pn_fir_tau attention over the 8-bit cache.
//
//   u_j = relu(scale q.k_j - tau), P_j = u_j^10, M = max_j u_j
//   O   = M / (M + gamma) * sum_j P_j v_j / (sum_j P_j + 1e-12)       over the keys j that the row sees
//
// A wave takes 64 keys at a time: four blocks of 16 tokens.  With the keys as rows of the first product and the
// queries as its columns, and key 16 g + 4 t + i as row 4 g + i of product t, lane group g gets all 16 scores of block
// g for its query, which is what the second product wants from it (the weights as columns, V^T as rows): scores go
// from one product to the other in registers, without LDS or exchange.  Key rows and value rows come straight from
// memory in 16-byte loads, the next tile's while this one is worked on.  Scales are powers of two, so e4m3 times scale
// is exact in bf16, and a block's key scale is one factor on its lane group's scores.
//
// A unit of work is a sequence, a key head and 16 NT rows (the query heads that share the key head, times query
// tokens).  A wave has a piece of one, which it finds by itself, as only the device knows the lengths; a second kernel
// joins the pieces.  Short caches, and calls with enough units to fill the card evenly, do without: a workgroup of four
// waves has a unit, takes its tiles in turn and adds up through LDS.  Of many rows, four waves have row tiles of their own
// and share the keys and values, in LDS.
//
// The powers are taken of u 2^-e with one e a row: 0 or, where a row's first scores are below 1/4, less; raised (and the
// sums scaled, exactly) when a score passes 2 2^e.  So weights stay below 2^10, and those down to 2^-100 of the
// largest are within fp32; values are summed with them as they are, so that 2^117 over the number of keys is the largest
// that cannot overflow.  With 2^8 in place of 2 it would be 2^47, and no faster.  e is -60 at least, for which keys of up to
// 2^60 (their scale times 2^60) and scores of up to 2^67 stay within fp32.
//
// bf16 queries: the weights are rounded to bf16 for the product and the same rounded values are summed, as the dense
// kernels do.  fp32 queries: queries and weights as three bf16 parts each (24 bits), keys and values are exact in one.
#pragma once

#include "cache.h"
#include "tiles_bf16.h"

#include <cmath>

namespace pnfx {

struct Header {  // of a piece, for the join: its unit, which of how many it is
  int b, h, rt, piece, n;
};

struct AttnArgs {
  Cache c;
  Span span;
  const void* q;
  void* o;
  int64_t qsb, qsh, qsn, osb, osh, osn;
  const float* tau;
  float scale, gamma;
  int has_gamma, causal, vec;  // vec: query rows of whole 8-byte parts, heads of whole 8 elements
  int G, R;           // query heads of a key head, row tiles
  int slots;          // waves that the card has room for
  // Of the pieces: how many there are, headers, [items][slot_rows][D] sums and [items][3][slot_rows]: the weights' sum,
  // peak, exponent
  int* items;
  Header* headers;
  float *acc, *stats;
  int slot_rows, most_items, join_waves;
};

// How a call is cut: row tiles of 16 NT rows, R for each sequence and key head; items: the most pieces of row tiles that units
// are cut into (0: one workgroup a unit); join_waves: that join a piece's part; bytes of workspace.
struct AttnPlan {
  bool shared;  // workgroups of four waves share their keys through LDS, in units of four row tiles
  int NT, R, slots, slot_rows, join_waves;
  int64_t units, items, header_bytes, acc_bytes, stat_bytes;
  int64_t bytes() const { return header_bytes + acc_bytes + stat_bytes; }
};

// Waves of a kernel that a SIMD holds, by its registers: the card has 1024 times as many slots.  In us with 1, 2, 3 and 4
// waves, the rule's own in brackets; one: a token of 64 sequences and 8 heads behind 500 MB of cache (NT = 1), rows: 100
// tokens of 8 sequences and 16 heads behind 4096 (NT = 2 up to 128 columns, else 1):
//   bf16   16, one 276 200 170 [161], rows 50 39 40 [42];   32, 162 100 84 [85], 54 41 [41] 52;   64, 110 85 [86] 86,
//   60 [50] 61 202;   80, 126 [97] 148 265, [77] 72 250 406;   128, 106 [90] 258 371, [94] 282 637 857;   144, [101] 135 301
//   424, [130] 136 521 774;   256, [94] 305 420 630, [216] 921 1390 2197
//   fp32   16, 336 231 202 [193], 65 56 57 [81];   32, 162 125 110 [108], 71 [60] 61 100;   64, 116 [90] 91 126, 88 [75] 139 355;
//   80, 122 [103] 246 401, [110] 195 462 729;   112, 111 [142] 331 474, [134] 359 718 1080;   128, 100 [153] 329 470,
//   [145] 444 924 1253;   256, [123] 372 549 735, [310] 1101 2004 2423
// The rule counts bf16's registers.  fp32's operands take three times as many: heads of 112 and 128 spill 80 and 110 of them
// with two waves (one token) where one wave would be faster, 16 columns 133 with four (many rows).
constexpr int resident(int bytes, int D, int NT) {
  return D * NT <= 32 ? 4 : bytes == 2 && D * NT <= 64 ? 3 : D * NT <= 128 ? 2 : 1;
}
// The same of the kernel whose waves share their keys: 256 times as many workgroups.  512 query tokens behind 7680, 2
// sequences of 16 heads, with 1, 2 and 3 (us): heads of 80 164, 107, 116; 96 160, 108, 131; 112 189, 117, 218; 128 201, 120,
// 233, although 32 and 109 registers spill with two in heads of 112 and 128, none with one.
constexpr int RESIDENT_SHARED = 2;

// The kernels, by the type of the queries and the head size in the cache.
int attn_bf16_64(const AttnArgs& a, const AttnPlan& p, hipStream_t st);    // up to 64
int attn_bf16_128(const AttnArgs& a, const AttnPlan& p, hipStream_t st);   // up to 128
int attn_bf16_256(const AttnArgs& a, const AttnPlan& p, hipStream_t st);
int attn_f32_64(const AttnArgs& a, const AttnPlan& p, hipStream_t st);
int attn_f32_128(const AttnArgs& a, const AttnPlan& p, hipStream_t st);
int attn_f32_256(const AttnArgs& a, const AttnPlan& p, hipStream_t st);

namespace {

typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int TILE = 64;  // keys that a wave takes at a time
constexpr int E_LAST = 120;  // 2^-120 u is below 2^8 for every fp32 u
constexpr int E_LEAST = -60, E_NONE = -100;  // of a row without scores, once it is joined
constexpr float TOP = 2.0f, LOW = 0.25f;

// Keys that a row tile's last row sees, from which its tiles follow.
template <int NT>
__device__ __forceinline__ int seen_by(const AttnArgs& a, int64_t start, int n, int rt) {
  if (start < 0 || start + n > a.c.capacity()) return 0;  // such sequences get NaN
  const int i0 = rt * 16 * NT / a.G, i1 = min((rt * 16 * NT + 16 * NT - 1) / a.G, n - 1);
  if (i0 >= n) return 0;
  return (int)(start + (a.causal ? i1 + 1 : n));
}
__device__ __forceinline__ int tiles_of(int seen) { return max(1, (seen + TILE - 1) / TILE); }

template <int DT>
struct Parts {  // how a head's columns fall on loads: whole 64, then 32, then 16, a quarter of each a lane group
  static constexpr int N64 = DT / 64, N32 = DT % 64 / 32, N16 = DT % 32 / 16;
  static constexpr int FRAGS = 2 * N64 + N32 + N16;
  // First of the 8 (N16: 4) columns of lane group g in fragment f.
  static __device__ __forceinline__ int col(int f, int g) {
    return f < 2 * N64 ? 64 * (f / 2) + 16 * g + 8 * (f % 2) : N32 && f == 2 * N64 ? 64 * N64 + 8 * g : 64 * N64 + 32 * N32 + 4 * g;
  }
};

template <int DT>
struct Raw {  // a tile of 64 keys and values as it lies in memory
  using P = Parts<DT>;
  u32x4 k64[4][P::N64 ? P::N64 : 1];  // vectors, so that a loop holds the loads' own registers, not copies of them
  u32x2 k32[4];
  unsigned k16[4];
  u32x4 v[DT / 16];
  float ks, vs;  // scales of block g; NaN where there is no such page
};

__device__ __forceinline__ bf16x8 eight(unsigned lo, unsigned hi, float s) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, s, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, s, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, s, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, s, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The high bits of those of four e4m3 numbers that are not finite: 0x7f of either sign, and under the largest scale,
// 2^120, from 0x78 (256) on.
__device__ __forceinline__ unsigned not_finite(unsigned w, float scale) {
  return ((w & 0x7f7f7f7fu) + (scale < two_to(120) ? 0x01010101u : 0x08080808u)) & 0x80808080u;
}

// What the weighted sum of a row is multiplied by: gate / (sum + 1e-12), both sums in units of 2^(10 e).  A row without
// scores has the gate 0, whatever fp32 makes of a small gamma.
__device__ __forceinline__ float factor(const AttnArgs& a, float z, float m, int e) {
  const float peak = ldexpf(m, e);
  const float gate = !a.has_gamma ? 1.0f : peak > 0 ? peak / (peak + a.gamma) : 0.0f;
  return gate / (z + ldexpf(1e-12f, -10 * e));
}

// What all lanes hold the same, as a scalar.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return (int64_t)((uint64_t)(unsigned)uniform((int)(x >> 32)) << 32 | (unsigned)uniform((int)x));
}

// WAVES waves with the same rows, each with every WAVES-th tile.
template <typename T, int DT, int NT, int WAVES>
struct Unit {
  static constexpr int STEP = WAVES * TILE;
  static constexpr bool ONCE = NT == 1 && DT <= 128;  // a call of up to 16 rows: one row tile
  static constexpr int FRAGS = Parts<DT>::FRAGS, ND = DT / 16, TERMS = sizeof(T) == 4 ? 3 : 1;
  const AttnArgs& a;
  int lane, wave, g, r16, b, h, rt, n;
  int64_t start;
  bf16x8 q[NT][FRAGS][TERMS];
  f32x4 acc[NT][ND];
  f32x4 z[NT];  // the weights' sum, the same four times
  float m[NT], unit[NT], off[NT];  // peak (of u 2^-e), scale 2^-e, -tau 2^-e
  bf16x8 ones;
  int e[NT], lim[NT];
  int min_lim;

  __device__ __forceinline__ Unit(const AttnArgs& args) : a(args) {
    lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), g = lane >> 4, r16 = lane & 15;
    for (int x = 0; x < 8; ++x) ones[x] = (bf16)1.0f;
  }
  __device__ __forceinline__ int row(int nt) const { return (rt * NT + nt) * 16 + r16; }
  // The lane number and the head size anew, so that what a unit's begin and end compute from them is not held in
  // registers (or spilled) over the tiles between.
  __device__ __forceinline__ int anew() {
    int d = a.c.d;
    asm volatile("" : "+v"(lane), "+s"(d));
    g = lane >> 4, r16 = lane & 15;
    return d;
  }

  __device__ __forceinline__ void begin(int b_, int h_, int rt_) {
    b = b_, h = h_, rt = rt_;
    const int d = anew();
    start = a.span.first(b), n = a.span.count(b);
    const int i0 = rt * 16 * NT / a.G;
    min_lim = a.causal ? (int)min(start + i0 + 1, (int64_t)(1 << 30)) : seen_by<NT>(a, start, n, rt);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row(nt), i = r / a.G;
      // rows without a query token see what others see: what they get is not stored
      lim[nt] = a.causal && i < n ? (int)(start + i + 1) : (int)min(start + n, (int64_t)1 << 30);
      const int there = max(min(i, n - 1), 0);
      const T* src = static_cast<const T*>(a.q) + b * a.qsb + (h * a.G + r % a.G) * a.qsh + there * a.qsn;
#pragma unroll
      for (int f = 0; f < FRAGS; ++f) {
        const int width = Parts<DT>::N16 && f == FRAGS - 1 ? 4 : 8;
        float v[8] = {};
        query(v, src, Parts<DT>::col(f, g), width, d);
#pragma unroll
        for (int x = 0; x < 8; ++x)
#pragma unroll
          for (int t = 0; t < TERMS; ++t) {
            q[nt][f][t][x] = (bf16)v[x];
            v[x] -= (float)(bf16)v[x];
          }
      }
#pragma unroll
      for (int j = 0; j < ND; ++j) acc[nt][j] = f32x4{0, 0, 0, 0};
      z[nt] = f32x4{0, 0, 0, 0}, m[nt] = 0, e[nt] = 0;
      rescale(nt);
    }
  }
  // Elements col .. col + width - 1 of a query row of d, zeros past its end.  (Loads within the row and masks: of a choice
  // between a load and zero the compiler makes a branch for each element, which took most of the time of calls with few
  // tiles.)
  __device__ __forceinline__ void query(float (&v)[8], const T* row, int col, int width, int d) const {
    if (a.vec) {  // whole 16 bytes, and no row ends inside 8 elements
      constexpr int EACH = 8 / sizeof(T);  // elements of 8 bytes
      const unsigned mask = col < d ? ~0u : 0u;
      const T* p = row + (col < d ? col : 0);
#pragma unroll
      for (int x = 0; x < 8; x += EACH) {
        if (x >= width) break;
        u32x2 w = *reinterpret_cast<const u32x2*>(p + x);
        w &= mask;
#pragma unroll
        for (int y = 0; y < EACH; ++y) {
          const unsigned u = w[sizeof(T) == 4 ? y : y / 2], bits = sizeof(T) == 4 ? u : y % 2 ? u & 0xffff0000u : u << 16;
          v[x + y] = __builtin_bit_cast(float, bits);
        }
      }
    } else {
#pragma unroll
      for (int x = 0; x < width; ++x) {
        const unsigned bits = __builtin_bit_cast(unsigned, to_f32(row[min(col + x, d - 1)]));
        v[x] = __builtin_bit_cast(float, col + x < d ? bits : 0u);
      }
    }
  }
  __device__ __forceinline__ void rescale(int nt) {
    const float s = two_to(-e[nt]);
    unit[nt] = a.scale * s, off[nt] = -a.tau[0] * s;
  }

  // Where a tile's blocks lie: that of the lane's key rows, and block g.  The table's numbers are asked for a tile
  // ahead of the rows that they name, before other loads, as loads come back in order.
  struct Pages {
    int k, v;
  };
  struct At {
    int k, v;
    bool there;
  };
  __device__ __forceinline__ Pages look(int key0) const {
    const int* t = a.c.table + b * a.c.table_rs;
    return Pages{t[min((key0 + 16 * (r16 >> 2)) >> a.c.page_shift, a.c.width - 1)],
                 t[min((key0 + 16 * g) >> a.c.page_shift, a.c.width - 1)]};
  }
  __device__ __forceinline__ int block(int id, int key) const {
    return ((((unsigned)id < (unsigned)a.c.pages ? id : 0) * a.c.H + h) << (a.c.page_shift - 4)) +
           ((key & (a.c.page - 1)) >> 4);
  }
  __device__ __forceinline__ At find(const Pages& p, int key0) const {
    return At{block(p.k, key0 + 16 * (r16 >> 2)), block(p.v, key0 + 16 * g), (unsigned)p.v < (unsigned)a.c.pages};
  }
  // Sixteen bytes of the cache.  What one row tile alone reads is not to be kept by the L2: 97.6 us against 110.6 for
  // the loads alone of 64 sequences of 4096 tokens, 16 heads of 64 (5.5 TB/s).
  static __device__ __forceinline__ u32x4 chunk(const uint8_t* p) {
    const u32x4* at = reinterpret_cast<const u32x4*>(p);
    return ONCE ? __builtin_nontemporal_load(at) : *at;
  }
  __device__ __forceinline__ void load_keys(const At& at, Raw<DT>& raw) const {
    using P = Parts<DT>;
    raw.ks = at.there ? two_to((int)a.c.k_scale[at.v] - 127) : __builtin_nanf("");
    const uint8_t* kb = a.c.k + (int64_t)at.k * (BLOCK * DT) + (r16 & 3) * DT;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint8_t* p = kb + 4 * t * DT;
#pragma unroll
      for (int i = 0; i < P::N64; ++i) raw.k64[t][i] = chunk(p + 64 * i + 16 * g);
      if (P::N32) raw.k32[t] = *reinterpret_cast<const u32x2*>(p + 64 * P::N64 + 8 * g);
      if (P::N16) raw.k16[t] = *reinterpret_cast<const unsigned*>(p + 64 * P::N64 + 32 * P::N32 + 4 * g);
    }
  }
  __device__ __forceinline__ void load_values(const At& at, Raw<DT>& raw) const {
    raw.vs = two_to(min((int)a.c.v_scale[at.v], 247) - 127);  // never written ones may be anything
    const uint8_t* vb = a.c.v + (int64_t)at.v * (BLOCK * DT) + r16 * 16;
#pragma unroll
    for (int j = 0; j < ND; ++j) raw.v[j] = chunk(vb + 256 * j);
  }
  __device__ __forceinline__ bf16x8 key_frag(const Raw<DT>& raw, int t, int f) const {
    using P = Parts<DT>;
    if (f < 2 * P::N64) {
      const u32x4 w = raw.k64[t][f / 2];
      return f % 2 ? eight(w[2], w[3], 1.0f) : eight(w[0], w[1], 1.0f);
    }
    if (P::N32 && f == 2 * P::N64) return eight(raw.k32[t][0], raw.k32[t][1], 1.0f);
    return eight(raw.k16[t], 0, 1.0f);
  }

  // A row whose scores pass 2 2^e, or whose first ones are all below 1/4: another e, the same for its four lane
  // groups, from the largest.
  __device__ __forceinline__ void another_e(float (&u)[16], float before, int nt) {
    const auto of_row = [](float x) {
      x = fmaxf(x, __shfl_xor(x, 16, 64));
      return fmaxf(x, __shfl_xor(x, 32, 64));
    };
    const float top = of_row(m[nt]), was = of_row(before);
    int up = E_LAST;  // of an infinite one
    if (top < __builtin_inff()) frexpf(top, &up);
    if (top > TOP) up = min(up, E_LAST - e[nt]);
    else if (was == 0 && top > 0 && top < LOW) up = max(up, E_LEAST);
    else return;
    const float f = was == 0 ? 1.0f : ldexpf(1.0f, -10 * up);
    z[nt] *= f, m[nt] = ldexpf(m[nt], -up), e[nt] += up;
#pragma unroll
    for (int j = 0; j < ND; ++j) acc[nt][j] *= f;
#pragma unroll
    for (int x = 0; x < 16; ++x) u[x] = ldexpf(u[x], -up);
    rescale(nt);
  }

  // u 2^-e of four of the lane's keys, from the product s.
  template <bool EDGE>
  __device__ __forceinline__ void scores(const f32x4& s, int nt, int t, float ks, int key0, float (&u)[16]) {
    const float c1 = ks * unit[nt];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = __builtin_elementwise_maximum(fmaf(s[i], c1, off[nt]), 0.0f);  // NaN stays
      if (EDGE) x = key0 + 16 * g + 4 * t + i < lim[nt] ? x : 0.0f;
      m[nt] = fmaxf(m[nt], x);
      u[4 * t + i] = x;
    }
  }
  // The weights of the lane's 16 keys, and their sum over all lane groups: a product with ones.
  __device__ __forceinline__ void weights(float (&u)[16], float before, int nt, bf16x8 (&p)[2][TERMS]) {
    const bool high = m[nt] > TOP && e[nt] < E_LAST, low = before == 0 && m[nt] > 0 && m[nt] < LOW;
    if (__builtin_expect(__any(high || low), 0)) another_e(u, before, nt);
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const float x2 = u[x] * u[x], x4 = x2 * x2;
      float w = x4 * x4 * x2;
#pragma unroll
      for (int k = 0; k < TERMS; ++k) {
        const bf16 r = (bf16)w;
        p[x / 8][k][x % 8] = r;
        w -= (float)r;
      }
    }
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int k = 0; k < TERMS; ++k) z[nt] = mfma16x16x32(ones, p[hf][k], z[nt]);
  }

  // One tile.  Its keys' and values' registers take the next tile's as soon as they have been used (`more`), so that
  // those loads are on their way over half of the work each.
  template <bool EDGE>
  __device__ __forceinline__ void tile(Raw<DT>& raw, int key0, bool more, Pages& next) {
    At at;
    float u[NT][16], before[NT];  // u 2^-e of the lane's 16 keys; m
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) before[nt] = m[nt];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f32x4 s[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int f = 0; f < FRAGS; ++f) {
        const bf16x8 kf = key_frag(raw, t, f);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < TERMS; ++i) s[nt] = mfma16x16x32(kf, q[nt][f][i], s[nt]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) scores<EDGE>(s[nt], nt, t, raw.ks, key0, u[nt]);
    }
    if (more) {
      at = find(next, key0 + STEP);
      next = look(key0 + 2 * STEP);
      load_keys(at, raw);
    }
    bf16x8 p[NT][2][TERMS];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) weights(u[nt], before[nt], nt, p[nt]);
    if (EDGE) values_edge(raw, key0);
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const bf16x8 v = value_frag(raw, j, hf);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < TERMS; ++i) acc[nt][j] = mfma16x16x32(v, p[nt][hf][i], acc[nt][j]);
      }
    if (more) load_values(at, raw);
  }
  __device__ __forceinline__ bf16x8 value_frag(const Raw<DT>& raw, int j, int hf) const {
    return eight(raw.v[j][2 * hf], raw.v[j][2 * hf + 1], raw.vs);
  }
  // In a tile that some row does not see whole, values that are not finite count as zeros, and a row that sees one gets
  // NaN there: a weight of zero would make NaN of them.
  __device__ __forceinline__ void values_edge(Raw<DT>& raw, int key0) {
    unsigned any = 0;
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) any |= not_finite(raw.v[j][i], raw.vs);
    if (__builtin_expect(!__any(any != 0), 1)) return;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      bf16x8 sees[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 8; ++x) sees[nt][x] = (bf16)(key0 + 16 * g + 8 * hf + x < lim[nt] ? 1.0f : 0.0f);
#pragma unroll
      for (int j = 0; j < ND; ++j) {
        const unsigned bl = not_finite(raw.v[j][2 * hf], raw.vs) >> 7, bh = not_finite(raw.v[j][2 * hf + 1], raw.vs) >> 7;
        raw.v[j][2 * hf] &= ~(bl * 0xff), raw.v[j][2 * hf + 1] &= ~(bh * 0xff);
        const bf16x8 bad = eight(bl * 0x38, bh * 0x38, 1.0f);  // 0x38: one
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const f32x4 hit = mfma16x16x32(bad, sees[nt], f32x4{0, 0, 0, 0});
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (hit[i] > 0) acc[nt][j][i] = __builtin_nanf("");
        }
      }
    }
  }

  // The tiles [t0, t1) of the unit.
  __device__ __forceinline__ void run(int t0, int t1) {
    const int keys = min(seen_by<NT>(a, start, n, rt), t1 * TILE);
    int key0 = (t0 + wave) * TILE;
    if (key0 >= keys) return;
    Raw<DT> raw;
    Pages next = look(key0);
    const At at = find(next, key0);
    next = look(key0 + STEP);
    load_keys(at, raw), load_values(at, raw);
    // tiles that every row sees whole, and others behind them, come first
    for (; key0 + TILE <= min_lim && key0 + STEP < keys; key0 += STEP) tile<false>(raw, key0, true, next);
    for (; key0 < keys; key0 += STEP) tile<true>(raw, key0, key0 + STEP < keys, next);
  }

  // Adds up four waves' sums in wave 0, in a fixed order.
  struct Lds {
    float z[WAVES][16 * NT], m[WAVES][16 * NT];
    int e[WAVES][16 * NT];
    float slab[2][NT * ND * 4 * 64];
  };
  __device__ __forceinline__ void row_peaks() {  // of the four lane groups
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt] = fmaxf(m[nt], __shfl_xor(m[nt], 16, 64));
      m[nt] = fmaxf(m[nt], __shfl_xor(m[nt], 32, 64));
      if (m[nt] == 0) e[nt] = E_NONE;
    }
  }
  __device__ __forceinline__ void join(Lds& s) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      if (g == 0) s.z[wave][16 * nt + r16] = z[nt][0], s.m[wave][16 * nt + r16] = m[nt], s.e[wave][16 * nt + r16] = e[nt];
    __syncthreads();
    const bool used = row(0) < a.G * n;  // of the first row tile's columns: one query token needs few of 16
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      int top = E_NONE;
      for (int w = 0; w < WAVES; ++w) top = max(top, s.e[w][16 * nt + r16]);
      const float f = ldexpf(1.0f, 10 * (e[nt] - top));
#pragma unroll
      for (int j = 0; j < ND; ++j) acc[nt][j] *= f;
      float zs = 0, ms = 0;
      for (int w = 0; w < WAVES; ++w) {
        const int up = s.e[w][16 * nt + r16] - top;
        zs += s.z[w][16 * nt + r16] * ldexpf(1.0f, 10 * up);
        ms = fmaxf(ms, ldexpf(s.m[w][16 * nt + r16], up));
      }
      z[nt][0] = zs, m[nt] = ms, e[nt] = top;
    }
    if (wave >= 2) put(s.slab[wave - 2], used);
    __syncthreads();
    if (wave < 2) add(s.slab[wave], used);
    __syncthreads();
    if (wave == 1) put(s.slab[0], used);
    __syncthreads();
    if (wave == 0) add(s.slab[0], used);
  }
  __device__ __forceinline__ void put(float* slab, bool used) const {
    if (!used) return;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < ND; ++j)
        *reinterpret_cast<f32x4*>(slab + ((nt * ND + j) * 64 + lane) * 4) = acc[nt][j];
  }
  __device__ __forceinline__ void add(const float* slab, bool used) {
    if (!used) return;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < ND; ++j)
        acc[nt][j] += *reinterpret_cast<const f32x4*>(slab + ((nt * ND + j) * 64 + lane) * 4);
  }

  __device__ __forceinline__ bool refused() const { return start < 0 || start + n > a.c.capacity(); }
  __device__ __forceinline__ void store() {  // one wave, the whole unit
    const int d = anew();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row(nt), i = r / a.G;
      if (i >= a.span.N) continue;
      const float f = factor(a, z[nt][0], m[nt], e[nt]);
      T* to = static_cast<T*>(a.o) + b * a.osb + (h * a.G + r % a.G) * a.osh + i * a.osn;
#pragma unroll
      for (int j = 0; j < ND; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int col = 16 * j + 4 * g + x;
          float v = acc[nt][j][x] * f;
          if (refused()) v = __builtin_nanf("");
          if (i >= n) v = 0;  // no query token
          if (col < d) to[col] = from_f32<T>(v);
        }
    }
  }
  __device__ __forceinline__ void keep(int slot) {  // a piece of the unit
    anew();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = 16 * nt + r16;
      if (row(nt) >= a.G * n) continue;
      float* st = a.stats + (int64_t)slot * 3 * a.slot_rows + r;
      if (g == 0) st[0] = z[nt][0], st[a.slot_rows] = m[nt], st[2 * a.slot_rows] = (float)e[nt];
      float* to = a.acc + ((int64_t)slot * a.slot_rows + r) * DT + 4 * g;
#pragma unroll
      for (int j = 0; j < ND; ++j) *reinterpret_cast<f32x4*>(to + 16 * j) = acc[nt][j];
    }
  }
};

// Consecutive shares on one XCD (workgroups go to the eight in turn), where neighbouring row tiles find each other's
// keys in its L2.
__device__ __forceinline__ int64_t place(int64_t wg, int64_t n) {
  const int64_t each = n / 8, more = n % 8, x = wg % 8;
  return x * each + min(x, more) + wg / 8;
}

// One workgroup of four waves a unit.
template <typename T, int DT, int NT>
__global__ __launch_bounds__(256, resident(sizeof(T), DT, NT)) void unit_kernel(AttnArgs a) {
  using U = Unit<T, DT, NT, 4>;
  __shared__ typename U::Lds lds;
  U u(a);
  const int w = (int)place(blockIdx.x, gridDim.x), bh = w / a.R;
  u.begin(bh / a.c.H, bh % a.c.H, a.R - 1 - w % a.R);  // the longest first
  u.run(0, tiles_of(seen_by<NT>(a, u.start, u.n, u.rt)));
  u.row_peaks();
  u.join(lds);
  if (u.wave == 0) u.store();
}

// A workgroup's piece of a unit: the sequence, which of how many pieces its tiles are cut into, which of the sequence's
// units, and the number of the item of all items; -1: none.
struct Piece {
  int b, tiles, piece, n, in, item, items;
};

// Pieces of units.  A sequence's tiles are cut alike for all its units (`each` of them: heads and row tiles), into as many
// equal pieces as give every slot of the card its share; neighbouring items then have the same tokens
// of neighbouring heads, which lie side by side in the pages: 64 sequences of up to 8192 tokens of random length,
// 16 heads of 64, one token each, take 106 us, with shares cut through the line of all units 127.  Of many rows and few
// sequences this is coarse (4 sequences of 512 query tokens and 16 heads of 64: 256 units each, for 2048 slots): behind 7680
// tokens each a billion pairs take 0.50 ms, behind random numbers of up to 7680 0.63 to 0.87.
__device__ __forceinline__ Piece piece_of(const AttnArgs& a, int lane, int each, int most_items) {
  const auto tiles_of_sequence = [&](int b) {
    const int64_t start = a.span.first(b);
    const int n = a.span.count(b);
    return tiles_of(start < 0 || start + n > a.c.capacity() || n == 0 ? 0 : (int)(start + n));
  };
  const int per = (a.c.B + 63) / 64, b0 = lane * per, b1 = min(b0 + per, a.c.B);
  int64_t all = 0;
  for (int b = b0; b < b1; ++b) all += tiles_of_sequence(b);
  for (int o = 1; o < 64; o *= 2) all += __shfl_xor(all, o, 64);
  // With s tiles a piece there are at most all / s + B pieces, and half of B less as a rule.
  const float slots = (float)a.slots / each, room = fmaxf(slots - 0.5f * a.c.B, 0.6f * slots);
  int64_t s = max((int64_t)1, uniform((int64_t)ceilf((float)all / room)));
  const auto pieces_of = [&](int tiles) { return (int)((tiles + s - 1) / s); };
  int sum, items;  // pieces of the sequences up to the end of each lane's; items of all of them
  for (;; ++s) {   // (again only if fp32's rounding gave a piece more than there is room for)
    sum = 0;
    for (int b = b0; b < b1; ++b) sum += pieces_of(tiles_of_sequence(b));
    for (int o = 1; o < 64; o *= 2) {
      const int x = __shfl_up(sum, o, 64);
      if (lane >= o) sum += x;
    }
    items = uniform(__shfl(sum, 63, 64)) * each;
    if (items <= most_items) break;
  }
  // consecutive items on one XCD (workgroups go to the eight in turn)
  const int eighth = (items + 7) / 8, item = (int)blockIdx.x % 8 * eighth + (int)blockIdx.x / 8;
  if ((int)blockIdx.x / 8 >= eighth || item >= items) return Piece{0, 0, 0, 0, 0, -1, items};
  const int line = item / each, group = __builtin_ctzll(__ballot(sum > line));
  int piece = line - (group ? uniform(__shfl(sum, group - 1, 64)) : 0), b = group * per, tiles, n;
  for (;;) {
    tiles = tiles_of_sequence(b), n = pieces_of(tiles);
    if (piece < n) break;
    piece -= n, ++b;
  }
  return Piece{b, tiles, piece, n, item % each, item, items};
}

// One wave a piece.
template <typename T, int DT, int NT>
__global__ __launch_bounds__(64, resident(sizeof(T), DT, NT)) void piece_kernel(AttnArgs a) {
  Unit<T, DT, NT, 1> u(a);
  const Piece p = piece_of(a, u.lane, a.c.H * a.R, a.most_items);
  if (p.item < 0) return;
  const int h = p.in / a.R, rt = p.in % a.R;
  u.begin(p.b, h, rt);
  u.run((int)((int64_t)p.tiles * p.piece / p.n), (int)((int64_t)p.tiles * (p.piece + 1) / p.n));
  u.row_peaks();
  if (p.n == 1) u.store();
  else u.keep(p.item);
  if (u.lane == 0) a.headers[p.item] = Header{p.b, h, rt, p.piece, p.n};
  // those that no item has, for the join
  if (u.lane == 0 && p.item == p.items - 1) *a.items = p.items;
}

// Many rows: a unit is four row tiles, a wave each, that share their keys and values.  Every wave brings a quarter of the
// next tile to LDS as the fragments that all of them read, in the order of their lanes: the bytes are loaded and turned to
// bf16 once for 64 NT rows, not for 16 NT.  (Fragments read four ahead of their products: no faster with heads of 64 and 128,
// spills with 256, of which a wave's results alone are half of its registers.)
template <typename T, int DT, int NT>
struct Sharing : Unit<T, DT, NT, 1> {
  using U = Unit<T, DT, NT, 1>;
  using P = Parts<DT>;
  using U::a, U::lane, U::wave, U::g, U::r16, U::b, U::rt, U::n, U::start, U::q, U::acc, U::m, U::lim;
  static constexpr int FRAGS = U::FRAGS, ND = U::ND, TERMS = U::TERMS, KEYS = 4 * FRAGS;
  struct Tile {
    u32x4 frag[KEYS + 2 * ND][64];
    float ks[4];  // of the blocks
    int odd[4];   // at an edge: whether a wave's values are not all finite
  };
  struct Quarter {  // as Raw
    u32x4 k64[P::N64 ? P::N64 : 1], v[(ND + 3) / 4];
    u32x2 k32;
    unsigned k16;
    float ks, vs;
  };
  __device__ __forceinline__ Sharing(const AttnArgs& args) : U(args) {}

  __device__ __forceinline__ void ask(const typename U::At& at, Quarter& w) const {
    w.ks = at.there ? two_to((int)a.c.k_scale[at.v] - 127) : __builtin_nanf("");
    w.vs = two_to(min((int)a.c.v_scale[at.v], 247) - 127);
    const uint8_t* p = a.c.k + (int64_t)at.k * (BLOCK * DT) + ((r16 & 3) + 4 * wave) * DT;
#pragma unroll
    for (int i = 0; i < P::N64; ++i) w.k64[i] = *reinterpret_cast<const u32x4*>(p + 64 * i + 16 * g);
    if (P::N32) w.k32 = *reinterpret_cast<const u32x2*>(p + 64 * P::N64 + 8 * g);
    if (P::N16) w.k16 = *reinterpret_cast<const unsigned*>(p + 64 * P::N64 + 32 * P::N32 + 4 * g);
    const uint8_t* vb = a.c.v + (int64_t)at.v * (BLOCK * DT) + r16 * 16 + 256 * wave;
#pragma unroll
    for (int j = 0; j < ND; j += 4)
      if (j + 3 < ND || j + wave < ND) w.v[j / 4] = *reinterpret_cast<const u32x4*>(vb + 256 * j);
  }
  __device__ __forceinline__ void put(const Quarter& w, Tile& tile, bool edge) const {
    u32x4* keys = &tile.frag[wave * FRAGS][lane];
#pragma unroll
    for (int f = 0; f < FRAGS; ++f) {
      bf16x8 x;
      if (f < 2 * P::N64) {
        const u32x4 c = w.k64[f / 2];
        x = f % 2 ? eight(c[2], c[3], 1.0f) : eight(c[0], c[1], 1.0f);
      } else if (P::N32 && f == 2 * P::N64) {
        x = eight(w.k32[0], w.k32[1], 1.0f);
      } else {
        x = eight(w.k16, 0, 1.0f);
      }
      keys[64 * f] = __builtin_bit_cast(u32x4, x);
    }
    u32x4* values = &tile.frag[KEYS + 2 * wave][lane];
    unsigned any = 0;
#pragma unroll
    for (int j = 0; j < ND; j += 4)
      if (j + 3 < ND || j + wave < ND) {
        const u32x4 c = w.v[j / 4];
        values[64 * 2 * j] = __builtin_bit_cast(u32x4, eight(c[0], c[1], w.vs));
        values[64 * (2 * j + 1)] = __builtin_bit_cast(u32x4, eight(c[2], c[3], w.vs));
        if (edge)
#pragma unroll
          for (int i = 0; i < 4; ++i) any |= not_finite(c[i], w.vs);
      }
    if (wave == 0 && r16 == 0) tile.ks[g] = w.ks;
    if (edge && (any = __any(any != 0), lane == 0)) tile.odd[wave] = any;
  }

  template <bool EDGE>
  __device__ __forceinline__ void compute(const Tile& tile, int key0) {
    const float ks = tile.ks[g];
    float u[NT][16], before[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) before[nt] = m[nt];
    f32x4 s[NT];
    each<KEYS>(tile.frag, [&](int i, bf16x8 k) {
      const int t = i / FRAGS, f = i % FRAGS;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (f == 0) s[nt] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < TERMS; ++x) s[nt] = mfma16x16x32(k, q[nt][f][x], s[nt]);
        if (f == FRAGS - 1) U::template scores<EDGE>(s[nt], nt, t, ks, key0, u[nt]);
      }
    });
    bf16x8 p[NT][2][TERMS];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) U::weights(u[nt], before[nt], nt, p[nt]);
    const auto add = [&](int i, bf16x8 v) {
      const int j = i / 2, hf = i % 2;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < TERMS; ++x) acc[nt][j] = mfma16x16x32(v, p[nt][hf][x], acc[nt][j]);
    };
    if (EDGE && __builtin_expect(tile.odd[0] | tile.odd[1] | tile.odd[2] | tile.odd[3], 0)) {  // as values_edge
      typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
      each<2 * ND>(tile.frag + KEYS, [&](int i, bf16x8 v) {
        const u16x8 bits = __builtin_bit_cast(u16x8, v);
        const u16x8 bad = __builtin_bit_cast(u16x8, (bits & 0x7f80) == 0x7f80);
        const bf16x8 one = __builtin_bit_cast(bf16x8, bad & 0x3f80);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          bf16x8 sees;
#pragma unroll
          for (int x = 0; x < 8; ++x) sees[x] = (bf16)(key0 + 16 * g + 8 * (i % 2) + x < lim[nt] ? 1.0f : 0.0f);
          const f32x4 hit = mfma16x16x32(one, sees, f32x4{0, 0, 0, 0});
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (hit[x] > 0) acc[nt][i / 2][x] = __builtin_nanf("");
        }
        add(i, __builtin_bit_cast(bf16x8, bits & ~bad));
      });
    } else {
      each<2 * ND>(tile.frag + KEYS, add);
    }
  }
  // f of N fragments in turn.
  template <int N, typename F>
  __device__ __forceinline__ void each(const u32x4 (*frag)[64], F f) const {
#pragma unroll
    for (int i = 0; i < N; ++i) f(i, __builtin_bit_cast(bf16x8, frag[i][lane]));
  }

  // The tiles [t0, t1) of the unit; all four waves come here together.
  __device__ __forceinline__ void run(int t0, int t1, Tile (&lds)[2]) {
    const int keys = min(seen_by<4 * NT>(a, start, n, rt / 4), t1 * TILE), mine = min(seen_by<NT>(a, start, n, rt), keys);
    // from here on, a tile is one that some row of the unit does not see whole
    const int whole = a.causal ? (int)min(start + rt / 4 * (64 * NT) / a.G + 1, (int64_t)(1 << 30)) : keys;
    int key0 = t0 * TILE;
    if (key0 >= keys) return;
    Quarter w;
    typename U::Pages next = U::look(key0);
    typename U::At at = U::find(next, key0);
    next = U::look(key0 + TILE);
    ask(at, w), put(w, lds[0], key0 + TILE > whole);
    at = U::find(next, key0 + TILE), next = U::look(key0 + 2 * TILE);  // beside the keys: some page of the sequence
    if (key0 + TILE < keys) ask(at, w);
    __syncthreads();
    for (int i = 0; key0 < keys; key0 += TILE, i ^= 1) {
      if (key0 < mine) {
        if (key0 + TILE > whole) compute<true>(lds[i], key0);
        else compute<false>(lds[i], key0);
      }
      if (key0 + TILE < keys) {
        put(w, lds[i ^ 1], key0 + 2 * TILE > whole);
        at = U::find(next, key0 + 2 * TILE), next = U::look(key0 + 3 * TILE);
        if (key0 + 2 * TILE < keys) ask(at, w);
      }
      __syncthreads();
    }
  }
};

template <typename T, int DT, int NT>
__global__ __launch_bounds__(256, RESIDENT_SHARED) void shared_kernel(AttnArgs a) {
  using S = Sharing<T, DT, NT>;
  __shared__ typename S::Tile lds[2];
  S u(a);
  const int R = a.R / 4;
  if (!a.most_items) {  // a workgroup a unit, the longest first
    const int w = (int)place(blockIdx.x, gridDim.x), bh = w / R;
    u.begin(bh / a.c.H, bh % a.c.H, 4 * (R - 1 - w % R) + u.wave);
    u.run(0, 1 << 24, lds);
    u.row_peaks();
    u.store();
    return;
  }
  const Piece p = piece_of(a, u.lane, a.c.H * R, a.most_items / 4);
  if (p.item < 0) return;
  const int h = p.in / R, rt = 4 * (p.in % R) + u.wave;
  u.begin(p.b, h, rt);
  u.run((int)((int64_t)p.tiles * p.piece / p.n), (int)((int64_t)p.tiles * (p.piece + 1) / p.n), lds);
  u.row_peaks();
  if (p.n == 1) u.store();
  else u.keep(4 * p.item + u.wave);
  if (u.lane == 0) a.headers[4 * p.item + u.wave] = Header{p.b, h, rt, p.piece, p.n};
  if (threadIdx.x == 0 && p.item == p.items - 1) *a.items = 4 * p.items;
}

// Joins the units that were cut: the waves of a unit's n pieces, a.join_waves for each, have equal parts of its results.
// A lane has a result and, where there are fewer results than lanes, every so many of the pieces; it goes over them once,
// the sums in units of the largest e so far, so that no load waits for another.
// Q: columns of a lane, 4 or, where the head size is no multiple of it, 1.
template <typename T, int DT, int NT, int Q>
__device__ __forceinline__ void join_part(const AttnArgs& a, const Header& u, int item, int part_wave, int lane) {
  constexpr int ROWS = 16 * NT;
  typedef float vec __attribute__((ext_vector_type(Q)));
  const int each = a.c.H * a.R, me = u.piece * a.join_waves + part_wave, wide = a.c.d / Q;
  const int count = a.span.count(u.b);
  const int rows = min(ROWS, a.G * a.span.N - u.rt * ROWS), live = min(rows, a.G * count - u.rt * ROWS);
  const int64_t start = a.span.first(u.b);
  const bool refused = start < 0 || start + count > a.c.capacity();
  // no part of less than 16 results: pieces come in lines of the cache
  const int all = rows * wide, parts = min(u.n * a.join_waves, max(1, all * Q / 16));
  if (me >= parts) return;
  const int x0 = (int)((int64_t)all * me / parts), x1 = (int)((int64_t)all * (me + 1) / parts);
  int width = 1;  // results at a time
  while (width < 64 && width < x1 - x0) width *= 2;
  for (int base = x0; base < x1; base += width) {
    const int x = base + (lane & (width - 1)), r = x / wide, c = x % wide * Q;
    float top = E_NONE, z = 0, m = 0;
    vec v = 0;
    const auto add = [&](float e, float z1, float m1, const vec& v1) {
      const float to = fmaxf(top, e);
      const int was = (int)(top - to), is = (int)(e - to);
      const float fw = ldexpf(1.0f, 10 * was), fi = ldexpf(1.0f, 10 * is);
      z = z * fw + z1 * fi, v = v * fw + v1 * fi, m = fmaxf(ldexpf(m, was), ldexpf(m1, is)), top = to;
    };
    if (x < x1 && r < live) {
#pragma unroll 8
      for (int i = lane / width; i < u.n; i += 64 / width) {
        const int64_t slot = item + (i - u.piece) * each;
        const float* st = a.stats + slot * 3 * a.slot_rows + r;
        add(st[2 * a.slot_rows], st[0], st[a.slot_rows],
            *reinterpret_cast<const vec*>(a.acc + (slot * a.slot_rows + r) * DT + c));
      }
    }
    for (int o = width; o < 64; o *= 2) {
      vec other;
#pragma unroll
      for (int y = 0; y < Q; ++y) other[y] = __shfl_xor((float)v[y], o, 64);
      add(__shfl_xor(top, o, 64), __shfl_xor(z, o, 64), __shfl_xor(m, o, 64), other);
    }
    if (lane < width && x < x1) {
      const float f = factor(a, z, m, (int)top);
      const int row = u.rt * ROWS + r;
      T* to = static_cast<T*>(a.o) + u.b * a.osb + (u.h * a.G + row % a.G) * a.osh + row / a.G * a.osn + c;
#pragma unroll
      for (int y = 0; y < Q; ++y) {
        float w = r < live ? v[y] * f : 0.0f;  // no query token: zero
        if (refused && r < live) w = __builtin_nanf("");
        to[y] = from_f32<T>(w);
      }
    }
  }
}
template <typename T, int DT, int NT>
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a) {
  const int wave = blockIdx.x * 4 + uniform((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int item = wave / a.join_waves, items = *a.items;
  const Header u = a.headers[min(item, a.most_items - 1)];
  if (item >= items || u.n == 1) return;
  if (a.c.d % 4 == 0) join_part<T, DT, NT, 4>(a, u, item, wave % a.join_waves, lane);
  else join_part<T, DT, NT, 1>(a, u, item, wave % a.join_waves, lane);
}

template <typename T, int DT, int NT>
int join(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
  join_kernel<T, DT, NT><<<dim3((unsigned)((p.items * p.join_waves + 3) / 4)), dim3(256), 0, st>>>(a);
  return launch_status("cached_attn");
}
template <typename T, int DT, int NT>
int run(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
  if (!p.items) {
    unit_kernel<T, DT, NT><<<dim3((unsigned)p.units), dim3(256), 0, st>>>(a);
    return launch_status("cached_attn");
  }
  piece_kernel<T, DT, NT><<<dim3((unsigned)p.items), dim3(64), 0, st>>>(a);
  if (int rc = launch_status("cached_attn")) return rc;
  return join<T, DT, NT>(a, p, st);
}
template <typename T, int DT, int NT>
int run_shared(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
  shared_kernel<T, DT, NT><<<dim3((unsigned)(p.items ? p.items / 4 : p.units)), dim3(256), 0, st>>>(a);
  const int rc = launch_status("cached_attn");
  return rc || !p.items ? rc : join<T, DT, NT>(a, p, st);
}
template <typename T, int DT>
int run_rows(const AttnArgs& a, const AttnPlan& p, hipStream_t st) {
  if constexpr (sizeof(T) == 2 && DT <= 128) {
    if (p.shared) return run_shared<T, DT, 2>(a, p, st);
  }
  if constexpr (DT <= 128) {
    if (p.NT == 2) return run<T, DT, 2>(a, p, st);
  }
  return run<T, DT, 1>(a, p, st);
}

}  // namespace
}  // namespace pnfx
