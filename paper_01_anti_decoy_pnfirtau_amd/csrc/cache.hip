// Writing the 8-bit key and value cache, and reading it back.
//
// Append.  One group of threads has the keys, or the values, of a block of 16 tokens of one sequence and head, one thread
// a column of the head: it holds the column's 16 tokens, so the FIR slides through registers, the largest |number| is a
// maximum over registers and then over the group, and the value block's row is one 16-byte store; the key block, whose
// rows are tokens, is turned through LDS and stored likewise.
//   k~_t = sum_j taps[j] k_{t-K+1+j}     in 64 bits: an fp32 sum would land on the other side of a rounding border
//                                        every few hundred thousand numbers, a 64-bit one practically never does
//   E    = the smallest for which no finite |number| is above 448 2^E, at least the block's so far if it is begun
//   byte = e4m3(number / 2^E), ties to even; NaN for what is not finite
// The tokens a begun block already has are rounded again when its scale grows: exact except below 2^-6 2^E, as a
// power of two leaves the significant bits alone.
//
// A group has several blocks in a row and asks for the next one's tokens before it works on this one's; the FIR's window
// stays in registers.
//
// The keys before the FIR that the next call needs are in `raw`, position p at p % 16.  Whoever reads them (the first
// and, for want of tokens before it, the second block of a call) must have done so before they are overwritten: one
// group has both blocks, each thread reads and writes its own column only, and writes last.
#include "cache.h"

#include <cmath>

namespace pnfx {
namespace {

constexpr int THREADS = 256;
constexpr int EACH = 2;  // blocks of a group, at least 2: 4 x 16 heads x 8192 tokens of 64 take 70 us, with 4 73

struct AppendArgs {
  Cache c;
  Span span;
  const void *k, *v;
  int64_t ksb, ksh, ksn, vsb, vsh, vsn;
  const float* taps;
  int taps_rows, K;
  int groups;  // of a sequence and head, for keys as for values
  int64_t items;
};

// The exponent of the smallest scale for numbers up to top >= 0: 448 = 1.75 * 2^8.
__device__ __forceinline__ int need(float top) {
  const unsigned b = __builtin_bit_cast(unsigned, top);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffff) > 0x600000);
  return max(e, E_LOWEST);  // zero and what is below the normal numbers: far below
}

// x cut to 20 fraction bits, the lowest set if any bit behind it was: fp32 holds that exactly (what is below its normal
// numbers is below every scale), times powers of two as well, and its rounding to e4m3 is that of x itself, as is its
// place beside 1.75 * 2^n.  From 2^128 on: infinite.
__device__ __forceinline__ float cut(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint64_t hi = (b & 0xffffffff00000000ull) | ((uint64_t)((unsigned)b != 0) << 32);
  return (float)__builtin_bit_cast(double, hi);
}

// |x| <= 448, infinite or NaN: e4m3 has no infinity, both become NaN.
__device__ __forceinline__ unsigned e4m3x4(const float (&x)[4]) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], lo, true);
}
__device__ __forceinline__ float value(unsigned byte) { return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0); }

__device__ __forceinline__ unsigned byte_of(const uint4& w, int t) {
  const unsigned u[4] = {w.x, w.y, w.z, w.w};
  return u[t >> 2] >> (8 * (t & 3)) & 0xff;
}

// The threads of a group (GROUP, a power of two) wait for each other's LDS accesses; one wave's are in order.
template <int GROUP>
__device__ __forceinline__ void group_sync() {
  if (GROUP > 64) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}
template <int GROUP>
__device__ __forceinline__ int group_max(int x, int* lds) {
#pragma unroll
  for (int o = (GROUP < 64 ? GROUP : 64) / 2; o >= 1; o /= 2) x = max(x, __shfl_xor(x, o, 64));
  if (GROUP > 64) {
    const int wave = threadIdx.x >> 6, first = wave & ~(GROUP / 64 - 1);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[wave] = x;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < GROUP / 64; ++i) x = max(x, lds[first + i]);
  }
  return x;
}

// A column's 16 bytes with those of tokens t0 .. t1 - 1 from x inv, the kept ones before them over `again`.
__device__ __forceinline__ uint4 column(const float (&x)[BLOCK], float inv, uint4 old, int t0, int t1, float again) {
  unsigned out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) y[u] = x[4 * i + u] * inv;
    out[i] = e4m3x4(y);
  }
  if (t0 > 0 || t1 < BLOCK) {
    const unsigned was[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) y[u] = value(was[i] >> (8 * u) & 0xff) * again;
      const unsigned kept = e4m3x4(y);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const unsigned mask = 0xffu << (8 * u);
        const int t = 4 * i + u;
        out[i] = (out[i] & ~mask) | ((t < t0 ? kept : t < t1 ? out[i] : was[i]) & mask);
      }
    }
  }
  return uint4{out[0], out[1], out[2], out[3]};
}

// The largest finite |x| of tokens t0 .. t1 - 1.
__device__ __forceinline__ float largest(const float (&x)[BLOCK], int t0, int t1) {
  float top = 0;
  if (t0 == 0 && t1 == BLOCK) {
#pragma unroll
    for (int t = 0; t < BLOCK; ++t) top = fmaxf(top, fabsf(x[t]));  // NaN loses in the maximum
    if (__builtin_expect(__all(top < __builtin_inff()), 1)) return top;
    top = 0;
  }
#pragma unroll
  for (int t = 0; t < BLOCK; ++t) {
    const float a = fabsf(x[t]);
    if (t >= t0 && t < t1 && a < __builtin_inff()) top = fmaxf(top, a);
  }
  return top;
}

// KT: the window that the FIR's taps are at the end of; 0: no FIR.  GROUP: threads of a block, at least its columns.
template <typename T, int KT, int GROUP>
__global__ __launch_bounds__(THREADS) void append_kernel(AppendArgs a) {
  __shared__ int peaks[THREADS / 64];
  __shared__ uint4 turn[THREADS];  // a key block, 16 bytes a thread
  constexpr int HIST = KT ? KT - 1 : 0, PER = THREADS / GROUP;
  const Cache& c = a.c;
  int within = threadIdx.x / GROUP;
  if (GROUP >= 64) within = __builtin_amdgcn_readfirstlane(within);  // the same for a wave: rows by scalar addresses
  unsigned item = blockIdx.x * PER + within;
  const bool exists = item < (unsigned)a.items;
  if (!exists) item = 0;
  const bool keys = item % 2 == 0;
  const int j = (int)(item / 2 % (unsigned)a.groups);
  const int bh = (int)(item / 2 / (unsigned)a.groups), b = bh / c.H, h = bh % c.H;
  const int col = threadIdx.x & (GROUP - 1);
  const bool mine = col < c.d;  // a column of the head; the others up to D hold zeros
  const int64_t s = a.span.first(b);
  const int n = a.span.count(b);
  const bool fits = exists && n > 0 && s >= 0 && s + n <= c.capacity();
  const T* src = keys ? static_cast<const T*>(a.k) + b * a.ksb + h * a.ksh
                      : static_cast<const T*>(a.v) + b * a.vsb + h * a.vsh;
  const int64_t sn = keys ? a.ksn : a.vsn;
  const int at_col = mine ? col : 0;
  const unsigned mask = mine ? ~0u : 0u;
  T* raw = static_cast<T*>(c.raw) + (int64_t)bh * RAW * c.d + at_col;
  const int skip = KT == 7 ? 0 : KT - a.K;  // a shorter filter's taps are the window's last
  float tap[KT ? KT : 1];
#pragma unroll
  for (int u = 0; u < KT; ++u)
    tap[u] = u >= skip ? a.taps[(a.taps_rows > 1 ? (int64_t)h * a.K : 0) + u - skip] : 0.0f;
  // (a mask, as the compiler turns a choice of a load or zero into a branch for each, which waits for its load)
  const auto masked = [&](T x) {
    return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, to_f32(x)) & mask);
  };
  // The call's tokens i0 .. i0 + count - 1 of the column; what is beside them is some token of it.
  const auto load = [&](auto& x, int off, int i0, auto count) {
    if (i0 >= 0 && i0 + count() <= n) {  // rows by one step
      const T* at = src + i0 * sn + at_col;
#pragma unroll
      for (int t = 0; t < count(); ++t) x[off + t] = masked(at[t * sn]);
    } else {
#pragma unroll
      for (int t = 0; t < count(); ++t) x[off + t] = masked(src[min(max(i0 + t, 0), n - 1) * sn + at_col]);
    }
  };
  struct Whole { constexpr int operator()() const { return HIST + BLOCK; } };
  struct Next { constexpr int operator()() const { return BLOCK; } };
  // w: the column's numbers, for keys those before the block, too; the next block's are on their way meanwhile
  float w[HIST + BLOCK];
  int64_t pos0 = (s & ~(int64_t)(BLOCK - 1)) + (int64_t)j * EACH * BLOCK;
  if (fits && pos0 < s + n) {
    load(w, 0, (int)(pos0 - s) - HIST, Whole{});
    if (HIST && keys && pos0 - HIST < s) {  // the first block
#pragma unroll
      for (int t = 0; t < HIST + BLOCK - 1; ++t) {
        const int64_t pos = pos0 - HIST + t;
        if (pos < s) w[t] = pos >= 0 && s - pos < a.K && mine ? to_f32(raw[(pos & (RAW - 1)) * c.d]) : 0.0f;
      }
    }
  }
#pragma unroll
  for (int r = 0; r < EACH; ++r, pos0 += BLOCK) {
    if (GROUP >= 64 && pos0 >= s + n) break;  // the same for all that meet at a barrier
    const int t0 = (int)max((int64_t)0, s - pos0);
    const int t1 = (int)min((int64_t)BLOCK, s + n - pos0);
    const int64_t block = fits && t1 > t0 ? c.block_at(b, h, pos0) : -1;
    const bool live = block >= 0;
    const bool part = t0 > 0 || t1 < BLOCK;
    uint8_t* bytes = (keys ? c.k : c.v) + block * BLOCK * c.D;
    uint8_t* scale = (keys ? c.k_scale : c.v_scale) + block;
    uint4 out = {0, 0, 0, 0}, old = {0, 0, 0, 0};
    int was = 0, e = E_LOWEST;
    // the block's bytes so far and its scale: a value column's own, or 16 bytes of the key block to be turned
    if (live && part && col < c.D) old = *reinterpret_cast<const uint4*>(bytes + col * BLOCK);
    if (live && t0 > 0) was = min((int)*scale, 247) - 127;
    float next[BLOCK], x[BLOCK];
    if (r + 1 < EACH && fits && pos0 + BLOCK < s + n) load(next, 0, (int)(pos0 + BLOCK - s), Next{});
    if (live) {
      if (KT && keys) {
        double win[KT ? KT : 1];
#pragma unroll
        for (int u = 0; u < HIST; ++u) win[u] = (double)w[u];
#pragma unroll
        for (int t = 0; t < BLOCK; ++t) {
          win[(HIST + t) % (KT ? KT : 1)] = (double)w[HIST + t];
          double acc = 0;
#pragma unroll
          for (int u = 0; u < KT; ++u)
            if (KT == 7 || u >= skip) acc = fma((double)tap[u], win[(t + u) % (KT ? KT : 1)], acc);
          x[t] = cut(acc);
        }
      } else {
#pragma unroll
        for (int t = 0; t < BLOCK; ++t) x[t] = w[HIST + t];
      }
      e = need(largest(x, t0, t1));
    }
    e = group_max<GROUP>(e, peaks);
    if (t0 > 0) e = max(e, was);
    if (keys) {
      uint8_t* lds = reinterpret_cast<uint8_t*>(turn + (threadIdx.x & ~(GROUP - 1)));
      if (part) {  // the column's old bytes
        group_sync<GROUP>();
        if (live && col < c.D) turn[threadIdx.x] = old;
        group_sync<GROUP>();
        unsigned q[4] = {0, 0, 0, 0};
        if (live && col < c.D)
#pragma unroll
          for (int t = 0; t < BLOCK; ++t) q[t >> 2] |= (unsigned)lds[t * c.D + col] << (8 * (t & 3));
        old = uint4{q[0], q[1], q[2], q[3]};
      }
      if (live) out = column(x, two_to(-e), old, t0, t1, ldexpf(1.0f, was - e));
      group_sync<GROUP>();
      if (live && col < c.D)
#pragma unroll
        for (int t = 0; t < BLOCK; ++t) lds[t * c.D + col] = (uint8_t)byte_of(out, t);
      group_sync<GROUP>();
      out = turn[threadIdx.x];
    } else {
      if (GROUP > 64) {  // the barriers that the workgroup's key group waits at
        if (part) group_sync<GROUP>(), group_sync<GROUP>();
        group_sync<GROUP>(), group_sync<GROUP>();
      }
      if (live) out = column(x, two_to(-e), old, t0, t1, ldexpf(1.0f, was - e));
    }
    if (live && col < c.D) *reinterpret_cast<uint4*>(bytes + col * BLOCK) = out;
    if (live && col == 0) *scale = (uint8_t)(e + 127);
#pragma unroll
    for (int t = 0; t < HIST; ++t) w[t] = w[BLOCK + t];
#pragma unroll
    for (int t = 0; t < BLOCK; ++t) w[HIST + t] = next[t];
  }
  if (keys && c.raw && j == 0 && fits && mine)
    for (int t = max(0, n - RAW); t < n; ++t) raw[((s + t) & (RAW - 1)) * c.d] = src[t * sn + at_col];
}

struct ReadArgs {
  Cache c;
  const int* first;
  int64_t first_all, count;
  void *k, *v;
  int group, groups, vec;  // vec: rows of results in whole 16-byte parts
  int64_t items;
};

// One group of threads a block of 16 positions: threads take 16 columns of a key each, and a column of the values.
template <typename T>
__global__ __launch_bounds__(THREADS) void read_kernel(ReadArgs a) {
  const Cache& c = a.c;
  const int per = THREADS / a.group;
  const unsigned item = blockIdx.x * per + threadIdx.x / a.group;
  const int col = threadIdx.x & (a.group - 1);
  if (item >= (unsigned)a.items || col >= c.D) return;
  const int64_t bh = item / (unsigned)a.groups;
  const int b = (int)bh / c.H, h = (int)bh % c.H;
  const int64_t first = a.first ? a.first[b] : a.first_all;
  const int64_t pos0 = (first & ~(int64_t)(BLOCK - 1)) + (int64_t)(item % (unsigned)a.groups) * BLOCK;
  const bool there = pos0 >= 0 && pos0 < c.capacity();
  const int64_t block = there ? c.block_at(b, h, pos0) : -1;
  constexpr int VEC = 16 / sizeof(T);
  // beside the capacity: zeros; in a page that does not exist: NaN
  const float none = there ? __builtin_nanf("") : 0.0f;
  {
    const int parts = c.D / 16, t = col / parts, at = col % parts * 16;
    const int64_t row = pos0 + t - first;
    if (row >= 0 && row < a.count) {
      float x[16];
      if (block >= 0) {
        const uint4 w = *reinterpret_cast<const uint4*>(c.k + block * BLOCK * c.D + t * c.D + at);
        const float s = ldexpf(1.0f, c.k_scale[block] - 127);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = value(byte_of(w, i)) * s;
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = none;
      }
      T* to = static_cast<T*>(a.k) + (bh * a.count + row) * c.d + at;
      if (a.vec) {
#pragma unroll
        for (int i = 0; i < 16; i += VEC) {
          T part[VEC];
#pragma unroll
          for (int u = 0; u < VEC; ++u) part[u] = from_f32<T>(x[i + u]);
          if (at + i < c.d) *reinterpret_cast<uint4*>(to + i) = *reinterpret_cast<uint4*>(part);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (at + i < c.d) to[i] = from_f32<T>(x[i]);
      }
    }
  }
  if (col >= c.d) return;
  uint4 w = {0, 0, 0, 0};
  float s = 0;
  if (block >= 0) {
    w = *reinterpret_cast<const uint4*>(c.v + block * BLOCK * c.D + col * BLOCK);
    s = ldexpf(1.0f, c.v_scale[block] - 127);
  }
  T* to = static_cast<T*>(a.v) + bh * a.count * c.d + col;
#pragma unroll
  for (int t = 0; t < BLOCK; ++t) {
    const int64_t row = pos0 + t - first;
    if (row >= 0 && row < a.count) to[row * c.d] = from_f32<T>(block >= 0 ? value(byte_of(w, t)) * s : none);
  }
}

int group_of(int D) {  // threads a block: a power of two that holds its columns
  int g = 16;
  while (g < D) g *= 2;
  return g;
}

int grid_of(int64_t items, int group, const char* what, int64_t* grid) {
  *grid = (items * group + THREADS - 1) / THREADS;
  PNFX_REQUIRE(*grid * THREADS < (1ll << 32), "%s: %lld blocks in one call", what, (long long)items);
  return PNFX_OK;
}

template <typename T, int KT>
void append_group(const AppendArgs& a, int group, int64_t grid, hipStream_t st) {
  const auto go = [&](auto kernel) { kernel<<<dim3((unsigned)grid), dim3(THREADS), 0, st>>>(a); };
  switch (group) {
    case 16: return go(append_kernel<T, KT, 16>);
    case 32: return go(append_kernel<T, KT, 32>);
    case 64: return go(append_kernel<T, KT, 64>);
    case 128: return go(append_kernel<T, KT, 128>);
    default: return go(append_kernel<T, KT, 256>);
  }
}
template <typename T>
void append_any(const AppendArgs& a, int group, int64_t grid, hipStream_t st) {
  if (!a.taps) append_group<T, 0>(a, group, grid, st);
  else if (a.K == 7) append_group<T, 7>(a, group, grid, st);  // the framework's filters
  else append_group<T, 16>(a, group, grid, st);
}

}  // namespace
}  // namespace pnfx

extern "C" int pnfx_cache_append(const pnfx_cache* cache, const void* k, int64_t ksb, int64_t ksh, int64_t ksn,
                                 const void* v, int64_t vsb, int64_t vsh, int64_t vsn, int64_t N,
                                 const int32_t* start, int64_t start_all, const int32_t* counts, const float* taps,
                                 int64_t taps_rows, int K, int dtype, void* stream) {
  using namespace pnfx;
  AppendArgs a = {};
  if (int rc = cache_of(cache, "cache_append", &a.c)) return rc;
  PNFX_REQUIRE(k && v, "cache_append: null pointer");
  PNFX_REQUIRE(dtype == PNFX_F32 || dtype == PNFX_BF16, "cache_append: dtype %d", dtype);
  PNFX_REQUIRE(N >= 1 && N < (1ll << 31) - 64, "cache_append: N=%lld", (long long)N);
  PNFX_REQUIRE(start || (start_all >= 0 && start_all < (1ll << 31)), "cache_append: start %lld", (long long)start_all);
  PNFX_REQUIRE(!taps || (K >= 1 && K <= 16 && (taps_rows == 1 || taps_rows == cache->H)),
               "cache_append: %d taps in %lld rows", K, (long long)taps_rows);
  PNFX_REQUIRE(!taps || cache->raw, "cache_append: a FIR needs the cache's raw keys");
  a.span = Span{start, counts, (int)start_all, (int)N};
  a.k = k, a.v = v, a.ksb = ksb, a.ksh = ksh, a.ksn = ksn, a.vsb = vsb, a.vsh = vsh, a.vsn = vsn;
  a.taps = taps, a.taps_rows = (int)taps_rows, a.K = taps ? K : 1;
  const int group = group_of(a.c.D);
  const int64_t blocks = (N + 2 * BLOCK - 2) / BLOCK;  // a call may begin at a block's last token
  a.groups = (int)((blocks + EACH - 1) / EACH);
  a.items = 2ll * a.c.B * a.c.H * a.groups;
  int64_t grid;
  if (int rc = grid_of(a.items, group, "cache_append", &grid)) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == PNFX_F32) append_any<float>(a, group, grid, st);
  else append_any<bf16>(a, group, grid, st);
  return launch_status("cache_append");
}

extern "C" int pnfx_cache_read(const pnfx_cache* cache, const int32_t* first, int64_t first_all, int64_t count,
                               void* k, void* v, int dtype, void* stream) {
  using namespace pnfx;
  ReadArgs a = {};
  if (int rc = cache_of(cache, "cache_read", &a.c)) return rc;
  PNFX_REQUIRE(k && v, "cache_read: null pointer");
  PNFX_REQUIRE(dtype == PNFX_F32 || dtype == PNFX_BF16, "cache_read: dtype %d", dtype);
  PNFX_REQUIRE(count >= 1 && count < (1ll << 31) - 64, "cache_read: count=%lld", (long long)count);
  PNFX_REQUIRE(first || (first_all >= 0 && first_all < (1ll << 31)), "cache_read: first %lld", (long long)first_all);
  const int vec = 16 / (dtype == PNFX_F32 ? 4 : 2);
  a.first = first, a.first_all = first_all, a.count = count, a.k = k, a.v = v;
  a.vec = a.c.d % vec == 0 && ((reinterpret_cast<uintptr_t>(k)) & 15) == 0;
  a.group = group_of(a.c.D);
  a.groups = (int)((count + 2 * BLOCK - 2) / BLOCK);
  a.items = (int64_t)a.c.B * a.c.H * a.groups;
  int64_t grid;
  if (int rc = grid_of(a.items, a.group, "cache_read", &grid)) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == PNFX_F32) read_kernel<float><<<dim3((unsigned)grid), dim3(THREADS), 0, st>>>(a);
  else read_kernel<bf16><<<dim3((unsigned)grid), dim3(THREADS), 0, st>>>(a);
  return launch_status("cache_read");
}
