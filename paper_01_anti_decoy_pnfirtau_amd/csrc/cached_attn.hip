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
// The waves of a workgroup take every fourth tile of the same rows, so that a key is read once by the workgroup
// whatever its number of rows (16 NT: query heads that share the key head, times query tokens), and add up through
// LDS.  The work of a call, 256 keys of one unit (sequence, key head, row tile) a step, is cut into equal shares for
// a fixed number of workgroups, whatever the lengths, which only the device knows; a unit that several workgroups
// have pieces of is joined by a second kernel.
//
// The powers are taken of u 2^-e with one e a row, raised (and the sums scaled, exactly) only when a score passes
// 2^8 2^e: a power of ten of the tenth lies within fp32 for scores 2^8 above and 2^12 below.  bf16 queries: the
// weights are rounded to bf16 for the product and the same rounded values are summed, as the dense kernels do.  fp32
// queries: queries and weights as three bf16 parts each (24 bits), keys and values are exact in one.
#include "cache.h"
#include "tiles_bf16.h"

#include <cmath>

namespace pnfx {
namespace {

typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int THREADS = 256, WAVES = 4, TILE = 64, STEP = WAVES * TILE;
constexpr int E_FIRST = -60;  // of a row without scores: 2^60 u is finite for u up to 2^67, and larger ones raise it again
constexpr float TOP = 256.0f;

struct Header {  // of a workgroup's unfinished unit, for the join
  int b, h, rt, last;  // last: the last workgroup that has a piece of it; -1: none
};

struct AttnArgs {
  Cache c;
  Span span;
  const void* q;
  void* o;
  int64_t qsb, qsh, qsn, osb, osh, osn;
  const float* tau;
  float scale, gamma;
  int has_gamma, causal;
  int Hq, G, R;       // query heads, those of a key head, row tiles
  int shares;         // workgroups that share the call's steps; 0: one workgroup a unit
  Header* headers;
  float *acc, *stats;  // pieces: [2 shares][rows][D], and [2 shares][3][rows]: sum, peak, exponent
};

// Keys that a row tile's last row sees, from which its steps follow.
template <int NT>
__device__ __forceinline__ int seen_by(const AttnArgs& a, int64_t start, int n, int rt) {
  if (start < 0 || start + n > a.c.capacity()) return 0;  // such sequences get NaN
  const int i0 = rt * 16 * NT / a.G, i1 = min((rt * 16 * NT + 16 * NT - 1) / a.G, n - 1);
  if (i0 >= n) return 0;
  return (int)(start + (a.causal ? i1 + 1 : n));
}
__device__ __forceinline__ int steps_of(int seen) { return max(1, (seen + STEP - 1) / STEP); }

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
  uint4 k64[4][P::N64 ? P::N64 : 1];
  uint2 k32[4];
  unsigned k16[4];
  uint4 v[DT / 16];
  float ks, vs;  // scales of block g; NaN where there is no such page
};

__device__ __forceinline__ bf16x8 eight(unsigned lo, unsigned hi, float s) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, s, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, s, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, s, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, s, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <typename T, int DT, int NT>
struct Unit {
  static constexpr int FRAGS = Parts<DT>::FRAGS, ND = DT / 16, TERMS = sizeof(T) == 4 ? 3 : 1;
  const AttnArgs& a;
  int lane, wave, g, r16, b, h, rt, n, nd, key_row;
  int64_t start;
  bf16x8 q[NT][FRAGS][TERMS];
  f32x4 acc[NT][ND];
  float z[NT], m[NT], unit[NT], off[NT];  // sum, peak (of u 2^-e), scale 2^-e, -tau 2^-e
  int e[NT], lim[NT];
  int min_lim;

  __device__ __forceinline__ Unit(const AttnArgs& args) : a(args) {
    lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r16 = lane & 15;
    key_row = 16 * (r16 >> 2) + (r16 & 3);
    nd = a.c.D / 16;
  }
  __device__ __forceinline__ int row(int nt) const { return (rt * NT + nt) * 16 + r16; }

  __device__ __forceinline__ void begin(int b_, int h_, int rt_) {
    b = b_, h = h_, rt = rt_;
    start = a.span.first(b), n = a.span.count(b);
    const int i0 = rt * 16 * NT / a.G;
    min_lim = a.causal ? (int)min(start + i0 + 1, (int64_t)(1 << 30)) : seen_by<NT>(a, start, n, rt);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row(nt), i = r / a.G;
      // rows without a query token see what others see: what they get is not stored
      lim[nt] = a.causal && i < n ? (int)(start + i + 1) : (int)min(start + n, (int64_t)1 << 30);
      const T* src = static_cast<const T*>(a.q) + b * a.qsb + (h * a.G + r % a.G) * a.qsh + i * a.qsn;
#pragma unroll
      for (int f = 0; f < FRAGS; ++f) {
        const int col = Parts<DT>::col(f, g);
        const int width = Parts<DT>::N16 && f == FRAGS - 1 ? 4 : 8;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          float v = 0;
          if (i < n && x < width && col + x < a.c.d) v = to_f32(src[col + x]);
#pragma unroll
          for (int t = 0; t < TERMS; ++t) {
            q[nt][f][t][x] = (bf16)v;
            v -= (float)(bf16)v;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < ND; ++j) acc[nt][j] = f32x4{0, 0, 0, 0};
      z[nt] = 0, m[nt] = 0, e[nt] = E_FIRST;
      rescale(nt);
    }
  }
  __device__ __forceinline__ void rescale(int nt) {
    const float s = two_to(-e[nt]);
    unit[nt] = a.scale * s, off[nt] = -a.tau[0] * s;
  }

  struct At {  // where a tile's blocks lie: that of the lane's key rows, and block g
    int64_t k, v;
    bool there;
  };
  __device__ __forceinline__ int64_t block_at(int key, bool* there) const {
    const int page = min(key >> a.c.page_shift, a.c.width - 1);
    const int id = a.c.table[b * a.c.table_rs + page];
    *there = (unsigned)id < (unsigned)a.c.pages;
    return ((int64_t)(*there ? id : 0) * a.c.H + h) * (a.c.page >> 4) + ((key & (a.c.page - 1)) >> 4);
  }
  __device__ __forceinline__ At find(int key0) const {
    At at;
    bool unused;
    at.k = block_at(key0 + 16 * (r16 >> 2), &unused);
    at.v = block_at(key0 + 16 * g, &at.there);
    return at;
  }
  __device__ __forceinline__ void load(const At& at, Raw<DT>& raw) const {
    using P = Parts<DT>;
    const int D = a.c.D;
    // columns past the head's re-load its first ones: they meet zeros of the query, and what is not finite there
    // belongs to the same key
    const auto within = [&](int col) { return DT == 16 || DT == 32 || col < D ? col : 0; };
    const uint8_t* kb = a.c.k + at.k * BLOCK * D + (r16 & 3) * D;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint8_t* p = kb + 4 * t * D;
#pragma unroll
      for (int i = 0; i < P::N64; ++i) raw.k64[t][i] = *reinterpret_cast<const uint4*>(p + within(64 * i + 16 * g));
      if (P::N32) raw.k32[t] = *reinterpret_cast<const uint2*>(p + within(64 * P::N64 + 8 * g));
      if (P::N16) raw.k16[t] = *reinterpret_cast<const unsigned*>(p + within(64 * P::N64 + 32 * P::N32 + 4 * g));
    }
    const uint8_t* vb = a.c.v + at.v * BLOCK * D + r16 * 16;
#pragma unroll
    for (int j = 0; j < ND; ++j)
      if (j < nd) raw.v[j] = *reinterpret_cast<const uint4*>(vb + 256 * j);
    raw.ks = at.there ? two_to((int)a.c.k_scale[at.v] - 127) : __builtin_nanf("");
    raw.vs = two_to((int)a.c.v_scale[at.v] - 127);
  }
  __device__ __forceinline__ bf16x8 key_frag(const Raw<DT>& raw, int t, int f) const {
    using P = Parts<DT>;
    if (f < 2 * P::N64) {
      const uint4& w = raw.k64[t][f / 2];
      return f % 2 ? eight(w.z, w.w, 1.0f) : eight(w.x, w.y, 1.0f);
    }
    if (P::N32 && f == 2 * P::N64) return eight(raw.k32[t].x, raw.k32[t].y, 1.0f);
    return eight(raw.k16[t], 0, 1.0f);
  }

  __device__ __forceinline__ void tile(const Raw<DT>& raw, int key0) {
    const bool edge = key0 + TILE > min_lim;  // some row does not see all of it
    f32x4 s[NT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int f = 0; f < FRAGS; ++f) {
        const bf16x8 kf = key_frag(raw, t, f);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < TERMS; ++i) s[nt][t] = mfma16x16x32(kf, q[nt][f][i], s[nt][t]);
      }
    }
    bf16x8 p[NT][2][TERMS];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float u[4][4];
      for (;;) {
        const float c1 = raw.ks * unit[nt], c0 = off[nt];
        float top = m[nt];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = fmaf(s[nt][t][i], c1, c0);
            u[t][i] = __builtin_elementwise_maximum(x, 0.0f);  // NaN stays
            if (edge) u[t][i] = key0 + 16 * g + 4 * t + i < lim[nt] ? u[t][i] : 0.0f;
            top = fmaxf(top, u[t][i]);
          }
        const bool over = top > TOP && e[nt] < 120;
        if (!__any(over)) {
          m[nt] = top;
          break;
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));  // one e a row: that of its four lane groups' largest
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (top > TOP && e[nt] < 120) {
          int up;
          if (top < two_to(100)) frexpf(top, &up);
          else up = 100;
          up = min(up, 120 - e[nt]);
          const float f = ldexpf(1.0f, -10 * up);
          z[nt] *= f, m[nt] = ldexpf(m[nt], -up), e[nt] += up;
#pragma unroll
          for (int j = 0; j < ND; ++j) acc[nt][j] *= f;
          rescale(nt);
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = u[t][i], x2 = x * x, x4 = x2 * x2;
          float w = x4 * x4 * x2;
          if (TERMS == 1) {
            const bf16 r = (bf16)w;
            p[nt][t / 2][0][4 * (t % 2) + i] = r;
            z[nt] += (float)r;
          } else {
            z[nt] += w;
#pragma unroll
            for (int k = 0; k < TERMS; ++k) {
              const bf16 r = (bf16)w;
              p[nt][t / 2][k][4 * (t % 2) + i] = r;
              w -= (float)r;
            }
          }
        }
    }
    bool odd = false;
    if (edge) {  // what is not finite in a value that some row does not see must not reach that row
#pragma unroll
      for (int j = 0; j < ND; ++j)
        if (j < nd)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const bf16x8 v = value_frag(raw, j, hf);
#pragma unroll
            for (int x = 0; x < 8; ++x) odd |= !(fabsf((float)v[x]) < __builtin_inff());
          }
      odd = __any(odd);
    }
    if (odd) {
      values_edge(raw, p, key0);
      return;
    }
#pragma unroll
    for (int j = 0; j < ND; ++j)
      if (j < nd)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const bf16x8 v = value_frag(raw, j, hf);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < TERMS; ++i) acc[nt][j] = mfma16x16x32(v, p[nt][hf][i], acc[nt][j]);
        }
  }
  __device__ __forceinline__ bf16x8 value_frag(const Raw<DT>& raw, int j, int hf) const {
    return hf ? eight(raw.v[j].z, raw.v[j].w, raw.vs) : eight(raw.v[j].x, raw.v[j].y, raw.vs);
  }
  // A tile with values that are not finite and rows that do not see all of it: those values count as zeros, and a row
  // that sees one gets NaN there.
  __device__ __forceinline__ void values_edge(const Raw<DT>& raw, const bf16x8 (&p)[NT][2][TERMS], int key0) {
#pragma unroll
    for (int j = 0; j < ND; ++j)
      if (j < nd)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          bf16x8 v = value_frag(raw, j, hf), bad = zero_bf16x8();
#pragma unroll
          for (int x = 0; x < 8; ++x)
            if (!(fabsf((float)v[x]) < __builtin_inff())) v[x] = (bf16)0.0f, bad[x] = (bf16)1.0f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            bf16x8 sees = zero_bf16x8();
#pragma unroll
            for (int x = 0; x < 8; ++x)
              if (key0 + 16 * g + 8 * hf + x < lim[nt]) sees[x] = (bf16)1.0f;
            const f32x4 hit = mfma16x16x32(bad, sees, f32x4{0, 0, 0, 0});
#pragma unroll
            for (int i = 0; i < TERMS; ++i) acc[nt][j] = mfma16x16x32(v, p[nt][hf][i], acc[nt][j]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (hit[i] > 0) acc[nt][j][i] = __builtin_nanf("");
          }
        }
  }

  // The steps [s0, s1) of the unit, of which the wave has one tile each.
  __device__ __forceinline__ void run(int s0, int s1) {
    const int seen = seen_by<NT>(a, start, n, rt);
    const int keys = min(seen, s1 * STEP);
    int key0 = s0 * STEP + wave * TILE;
    if (key0 >= keys) return;
    Raw<DT> raw[2];
    load(find(key0), raw[0]);
    At next = find(key0 + STEP);
    for (;;) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (key0 + STEP < keys) {
          load(next, raw[1 - i]);
          next = find(key0 + 2 * STEP);
        }
        tile(raw[i], key0);
        key0 += STEP;
        if (key0 >= keys) return;
      }
    }
  }

  // Adds up the four waves' sums in wave 0, in a fixed order.
  struct Lds {
    float z[WAVES][16 * NT], m[WAVES][16 * NT];
    int e[WAVES][16 * NT];
    float slab[2][NT * ND * 4 * 64];
  };
  __device__ __forceinline__ void join(Lds& s) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int o = 16; o <= 32; o *= 2) {
        z[nt] += __shfl_xor(z[nt], o, 64);
        m[nt] = fmaxf(m[nt], __shfl_xor(m[nt], o, 64));
      }
      if (g == 0) s.z[wave][16 * nt + r16] = z[nt], s.m[wave][16 * nt + r16] = m[nt], s.e[wave][16 * nt + r16] = e[nt];
    }
    __syncthreads();
    const bool used = row(0) < a.G * n;  // of the first row tile's columns: one query token needs few of 16
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      int top = E_FIRST;
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
      z[nt] = zs, m[nt] = ms, e[nt] = top;
    }
    if (wave >= 2) put(s.slab[wave - 2], used);
    __syncthreads();
    if (wave < 2) add(s.slab[wave], used);
    __syncthreads();
    if (wave == 1) put(s.slab[0], used);
    __syncthreads();
    if (wave == 0) add(s.slab[0], used);
    __syncthreads();
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
  __device__ __forceinline__ void store() const {  // wave 0, the whole unit
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row(nt), i = r / a.G;
      if (i >= a.span.N) continue;
      const float f = factor(a, z[nt], m[nt], e[nt]);
      T* to = static_cast<T*>(a.o) + b * a.osb + (h * a.G + r % a.G) * a.osh + i * a.osn;
#pragma unroll
      for (int j = 0; j < ND; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int col = 16 * j + 4 * g + x;
          float v = acc[nt][j][x] * f;
          if (refused()) v = __builtin_nanf("");
          if (i >= n) v = 0;  // no query token
          if (col < a.c.d) to[col] = from_f32<T>(v);
        }
    }
  }
  __device__ __forceinline__ void keep(int slot) const {  // wave 0, a piece of the unit
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = 16 * nt + r16;
      if (row(nt) >= a.G * n) continue;
      float* st = a.stats + (int64_t)slot * 3 * 16 * NT + r;
      if (g == 0) st[0] = z[nt], st[16 * NT] = m[nt], st[2 * 16 * NT] = (float)e[nt];
      float* to = a.acc + ((int64_t)slot * 16 * NT + r) * DT + 4 * g;
#pragma unroll
      for (int j = 0; j < ND; ++j) *reinterpret_cast<f32x4*>(to + 16 * j) = acc[nt][j];
    }
  }
  // What the weighted sum of a row is multiplied by: gate / (sum + 1e-12), both sums in units of 2^(10 e).
  static __device__ __forceinline__ float factor(const AttnArgs& a, float z, float m, int e) {
    const float peak = ldexpf(m, e);
    const float gate = a.has_gamma ? peak / (peak + a.gamma) : 1.0f;
    return gate / (z + ldexpf(1e-12f, -10 * e));
  }
};

// Consecutive shares on one XCD (workgroups go to the eight in turn), where neighbouring row tiles find each other's
// keys in its L2.
__device__ __forceinline__ int64_t place(int64_t wg, int64_t n) {
  const int64_t each = n / 8, more = n % 8, x = wg % 8;
  return x * each + min(x, more) + wg / 8;
}

template <typename T, int DT, int NT>
__global__ __launch_bounds__(THREADS, DT * NT <= 128 ? 2 : 1) void attn_kernel(AttnArgs a) {
  __shared__ typename Unit<T, DT, NT>::Lds lds;
  Unit<T, DT, NT> u(a);
  if (!a.shares) {
    const int64_t id = place(blockIdx.x, gridDim.x);
    const int rt = a.R - 1 - (int)(id % a.R);  // the longest first
    const int64_t bh = id / a.R;
    u.begin((int)(bh / a.c.H), (int)(bh % a.c.H), rt);
    u.run(0, steps_of(seen_by<NT>(a, u.start, u.n, rt)));
    u.join(lds);
    if (u.wave == 0) u.store();
    return;
  }
  // The steps of all sequences before each of 256 groups of them
  __shared__ int64_t before[THREADS + 1];
  __shared__ int64_t wave_sum[WAVES];
  const int per = (a.c.B + THREADS - 1) / THREADS;
  const auto steps_of_sequence = [&](int b) {
    int64_t t = 0;
    const int64_t start = a.span.first(b);
    const int n = a.span.count(b);
    for (int rt = 0; rt < a.R; ++rt) t += steps_of(seen_by<NT>(a, start, n, rt));
    return t * a.c.H;
  };
  {
    int64_t mine = 0;
    for (int i = 0; i < per; ++i) {
      const int b = threadIdx.x * per + i;
      if (b < a.c.B) mine += steps_of_sequence(b);
    }
    int64_t sum = mine;
    for (int o = 1; o < 64; o *= 2) {
      const int64_t x = __shfl_up(sum, o, 64);
      if (u.lane >= o) sum += x;
    }
    if (u.lane == 63) wave_sum[u.wave] = sum;
    __syncthreads();
    for (int w = 0; w < u.wave; ++w) sum += wave_sum[w];
    before[threadIdx.x + 1] = sum;
    if (threadIdx.x == 0) before[0] = 0;
    __syncthreads();
  }
  const int64_t all = before[THREADS], share = (all + a.shares - 1) / a.shares;
  const int w = (int)place(blockIdx.x, gridDim.x);
  int64_t at = w * share;
  const int64_t end = min(all, at + share);
  if (threadIdx.x == 0) a.headers[w] = Header{0, 0, 0, -1};
  if (at >= end) return;
  int lo = 0, hi = THREADS;  // before[lo] <= at < before[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (before[mid] <= at) lo = mid;
    else hi = mid;
  }
  int64_t skip = at - before[lo];
  int b = lo * per;
  for (;;) {
    const int64_t t = steps_of_sequence(b);
    if (skip < t) break;
    skip -= t, ++b;
  }
  const int64_t head = steps_of_sequence(b) / a.c.H;
  int h = (int)(skip / head), rt = 0;
  skip %= head;
  for (;;) {
    const int t = steps_of(seen_by<NT>(a, a.span.first(b), a.span.count(b), rt));
    if (skip < t) break;
    skip -= t, ++rt;
  }
  while (at < end) {
    u.begin(b, h, rt);
    const int t = steps_of(seen_by<NT>(a, u.start, u.n, rt));
    const int s0 = (int)skip, s1 = (int)min((int64_t)t, s0 + end - at);
    u.run(s0, s1);
    u.join(lds);
    if (u.wave == 0) {
      if (s0 == 0 && s1 == t) u.store();
      else u.keep(2 * w + (s0 == 0));
      if (s0 == 0 && s1 < t && threadIdx.x == 0) a.headers[w] = Header{b, h, rt, (int)((at + t - 1) / share)};
    }
    at += s1 - s0, skip = 0;
    if (++rt == a.R) {
      rt = 0;
      if (++h == a.c.H) h = 0, ++b;
    }
  }
}

// Joins the pieces of the unit that workgroup w began and others went on with.
template <typename T, int DT, int NT>
__global__ __launch_bounds__(THREADS) void join_kernel(AttnArgs a) {
  const Header u = a.headers[blockIdx.x];
  if (u.last < 0) return;
  constexpr int ROWS = 16 * NT;
  const int first = 2 * blockIdx.x + 1, n = u.last - (int)blockIdx.x;  // slots first, first + 1, first + 3, ..
  const auto slot = [&](int i) { return (int64_t)(i == 0 ? first : first - 1 + 2 * i); };
  const int count = a.span.count(u.b);
  const int64_t start = a.span.first(u.b);
  const bool refused = start < 0 || start + count > a.c.capacity();
  for (int x = threadIdx.x; x < ROWS * a.c.d; x += THREADS) {
    const int r = x / a.c.d, col = x % a.c.d;
    const int row = u.rt * ROWS + r, i = row / a.G;
    if (i >= a.span.N) continue;
    float v = 0;
    if (i < count) {
      float top = E_FIRST;
      for (int s = 0; s <= n; ++s) top = fmaxf(top, a.stats[slot(s) * 3 * ROWS + 2 * ROWS + r]);
      float z = 0, m = 0;
      for (int s = 0; s <= n; ++s) {
        const float* st = a.stats + slot(s) * 3 * ROWS + r;
        const int up = (int)(st[2 * ROWS] - top);
        const float f = ldexpf(1.0f, 10 * up);
        z += st[0] * f, m = fmaxf(m, ldexpf(st[ROWS], up));
        v += a.acc[(slot(s) * ROWS + r) * DT + col] * f;
      }
      v *= Unit<T, DT, NT>::factor(a, z, m, (int)top);
      if (refused) v = __builtin_nanf("");
    }
    static_cast<T*>(a.o)[u.b * a.osb + (u.h * a.G + row % a.G) * a.osh + i * a.osn + col] = from_f32<T>(v);
  }
}

// --------------------------------------------------------------------------------------- host
int padded(int D) {  // head sizes that kernels are built for
  for (int x : {16, 32, 64, 96, 128})
    if (D <= x) return x;
  return 256;
}

struct Plan {
  int DT, NT, R, shares;
  int64_t units, header_bytes, acc_bytes, stat_bytes;
  int64_t bytes() const { return header_bytes + acc_bytes + stat_bytes; }
};

Plan plan_of(int64_t B, int64_t H, int64_t G, int64_t N, int D, int64_t capacity) {
  Plan p = {};
  p.DT = padded(D);
  const int64_t rows = G * N;
  p.NT = rows <= 16 ? 1 : 2;
  p.R = (int)((rows + 16 * p.NT - 1) / (16 * p.NT));
  p.units = B * H * p.R;
  const int64_t steps = (capacity + STEP - 1) / STEP;
  // One workgroup a unit where no cut can gain: short caches, whose few steps cost less than the join's launch, and
  // enough row tiles for the card to even out by itself.
  if (steps <= 2 || (p.R > 1 && p.units >= 2048)) return p;
  p.shares = (int)std::min<int64_t>(p.units * steps, 1024);
  const auto round = [](int64_t x) { return (x + 255) & ~(int64_t)255; };
  p.header_bytes = round(p.shares * (int64_t)sizeof(Header));
  p.acc_bytes = round(2ll * p.shares * 16 * p.NT * p.DT * 4);
  p.stat_bytes = round(2ll * p.shares * 3 * 16 * p.NT * 4);
  return p;
}

template <typename T, int DT, int NT>
int run(const AttnArgs& a, const Plan& p, hipStream_t st) {
  attn_kernel<T, DT, NT><<<dim3((unsigned)(p.shares ? p.shares : p.units)), dim3(THREADS), 0, st>>>(a);
  if (int rc = launch_status("cached_attn")) return rc;
  if (!p.shares) return PNFX_OK;
  join_kernel<T, DT, NT><<<dim3((unsigned)p.shares), dim3(THREADS), 0, st>>>(a);
  return launch_status("cached_attn");
}

template <typename T>
int run_any(const AttnArgs& a, const Plan& p, hipStream_t st) {
#define PNFX_CASE(DT) \
  case DT: return p.NT == 1 ? run<T, DT, 1>(a, p, st) : run<T, DT, 2>(a, p, st)
  switch (p.DT) {
    PNFX_CASE(16);
    PNFX_CASE(32);
    PNFX_CASE(64);
    PNFX_CASE(96);
    PNFX_CASE(128);
    PNFX_CASE(256);
  }
#undef PNFX_CASE
  return PNFX_EUNSUPPORTED;
}

}  // namespace
}  // namespace pnfx

extern "C" int64_t pnfx_cached_attn_workspace_size(const pnfx_cache* cache, int64_t Hq, int64_t N) {
  using namespace pnfx;
  Cache c;
  if (cache_of(cache, "cached_attn", &c) || N < 1 || Hq < c.H || Hq % c.H) return 0;
  return plan_of(c.B, c.H, Hq / c.H, N, c.D, c.capacity()).bytes();
}

extern "C" int pnfx_cached_attn(const pnfx_cache* cache, const void* q, int64_t qsb, int64_t qsh, int64_t qsn, void* o,
                                int64_t osb, int64_t osh, int64_t osn, int64_t Hq, int64_t N, const int32_t* start,
                                int64_t start_all, const int32_t* counts, const float* tau, float scale, float gamma,
                                int has_gamma, int causal, int dtype, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  using namespace pnfx;
  AttnArgs a = {};
  if (int rc = cache_of(cache, "cached_attn", &a.c)) return rc;
  PNFX_REQUIRE(q && o && tau, "cached_attn: null pointer");
  PNFX_REQUIRE(dtype == PNFX_F32 || dtype == PNFX_BF16, "cached_attn: dtype %d", dtype);
  PNFX_REQUIRE(Hq >= a.c.H && Hq % a.c.H == 0 && Hq < (1 << 20), "cached_attn: %lld query heads for %d key heads",
               (long long)Hq, a.c.H);
  PNFX_REQUIRE(N >= 1 && Hq / a.c.H * N < (1ll << 31) - 64, "cached_attn: N=%lld", (long long)N);
  PNFX_REQUIRE(start || (start_all >= 0 && start_all < (1ll << 31)), "cached_attn: start %lld", (long long)start_all);
  const Plan p = plan_of(a.c.B, a.c.H, Hq / a.c.H, N, a.c.D, a.c.capacity());
  PNFX_REQUIRE(p.units * THREADS < (1ll << 32), "cached_attn: %lld row tiles in one call", (long long)p.units);
  PNFX_REQUIRE(!p.bytes() || (workspace && workspace_bytes >= p.bytes() &&
                              (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
               "cached_attn: workspace needs %lld bytes, 16-byte aligned", (long long)p.bytes());
  a.span = Span{start, counts, (int)start_all, (int)N};
  a.q = q, a.o = o, a.qsb = qsb, a.qsh = qsh, a.qsn = qsn, a.osb = osb, a.osh = osh, a.osn = osn;
  a.tau = tau, a.scale = scale, a.gamma = gamma, a.has_gamma = has_gamma, a.causal = causal;
  a.Hq = (int)Hq, a.G = (int)Hq / a.c.H, a.R = p.R, a.shares = p.shares;
  char* ws = static_cast<char*>(workspace);
  a.headers = reinterpret_cast<Header*>(ws);
  a.acc = reinterpret_cast<float*>(ws + p.header_bytes);
  a.stats = reinterpret_cast<float*>(ws + p.header_bytes + p.acc_bytes);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return dtype == PNFX_F32 ? run_any<float>(a, p, st) : run_any<bf16>(a, p, st);
}
