// Writing the 8-bit key and value cache, and reading it back.
//
// Append.  One group of threads has a block of 16 tokens of one sequence and head, one thread a column of the head:
// it holds the column's 16 tokens, so the FIR slides through registers, the largest |number| is a maximum over
// registers and then over the group, and the value block's row is one 16-byte store.
//   k~_t = sum_j taps[j] k_{t-K+1+j}     in 64 bits: an fp32 sum would land on the other side of a rounding border
//                                        every few hundred thousand numbers, a 64-bit one practically never does
//   E    = the smallest for which no finite |number| is above 448 2^E, at least the block's so far if it is begun
//   byte = e4m3(number / 2^E), ties to even; NaN for what is not finite
// The tokens a begun block already has are rounded again when its scale grows: exact except below 2^-6 2^E, as a
// power of two leaves the significant bits alone.
//
// The keys before the FIR that the next call needs are in `raw`, position p at p % 16.  Whoever reads them (the first
// and the second block of a sequence's tokens) must have done so before they are overwritten: one group has both
// blocks, each thread reads and writes its own column only, and writes last.
#include "cache.h"

#include <cmath>

namespace pnfx {
namespace {

constexpr int THREADS = 256;

struct AppendArgs {
  Cache c;
  Span span;
  const void *k, *v;
  int64_t ksb, ksh, ksn, vsb, vsh, vsn;
  const float* taps;
  int taps_rows, K;
  int group, groups;  // threads a block, groups a sequence and head
  int64_t items;
};

// The exponent of the smallest scale for numbers up to top >= 0: 448 = 1.75 * 2^8.
__device__ __forceinline__ int need(double top) {
  const uint64_t b = __builtin_bit_cast(uint64_t, top);
  const int e = (int)(b >> 52) - 1023 - 8 + ((b & 0xfffffffffffffull) > 0xc000000000000ull);
  return max(e, E_LOWEST);  // zero and what is below the normal numbers: far below
}

// x as e4m3: the number is first cut to 20 fraction bits, the lowest set if any bit behind it was, from which fp32 is
// exact and the conversion's rounding that of x itself.
__device__ __forceinline__ float cut(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint64_t hi = (b & 0xffffffff00000000ull) | ((uint64_t)((unsigned)b != 0) << 32);
  return (float)__builtin_bit_cast(double, hi);
}
__device__ __forceinline__ unsigned e4m3(float x) {  // |x| <= 448, or NaN
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false) & 0xff;
}
__device__ __forceinline__ float value(unsigned byte) { return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0); }

__device__ __forceinline__ unsigned byte_of(const uint4& w, int t) {
  const unsigned u[4] = {w.x, w.y, w.z, w.w};
  return u[t >> 2] >> (8 * (t & 3)) & 0xff;
}

// Maximum over the threads of a group (a power of two of them).
__device__ __forceinline__ int group_max(int x, int group, int* lds) {
  for (int o = min(group, 64) >> 1; o >= 1; o >>= 1) x = max(x, __shfl_xor(x, o, 64));
  if (group > 64) {  // the same for the whole workgroup
    const int wave = threadIdx.x >> 6, first = wave & ~(group / 64 - 1);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[wave] = x;
    __syncthreads();
    for (int i = 0; i < group / 64; ++i) x = max(x, lds[first + i]);
  }
  return x;
}

// KT: the window that the FIR's taps are at the end of; 0: no FIR.
template <typename T, int KT>
__global__ __launch_bounds__(THREADS) void append_kernel(AppendArgs a) {
  __shared__ int lds[4];
  constexpr int HIST = KT ? KT - 1 : 0;
  const Cache& c = a.c;
  const int per = THREADS / a.group;
  int64_t item = (int64_t)blockIdx.x * per + threadIdx.x / a.group;
  const bool exists = item < a.items;
  if (!exists) item = 0;
  const int j = (int)(item % a.groups);
  const int h = (int)(item / a.groups % c.H), b = (int)(item / a.groups / c.H);
  const int col = threadIdx.x & (a.group - 1);
  const bool mine = exists && col < c.d;  // a column of the head; the others up to D hold zeros
  const int64_t s = a.span.first(b);
  const int n = a.span.count(b);
  const bool fits = exists && s >= 0 && s + n <= c.capacity();
  const T* k = static_cast<const T*>(a.k) + b * a.ksb + h * a.ksh + (mine ? col : 0);
  const T* v = static_cast<const T*>(a.v) + b * a.vsb + h * a.vsh + (mine ? col : 0);
  T* raw = static_cast<T*>(c.raw) + ((int64_t)b * c.H + h) * RAW * c.d + col;
  const int skip = KT == 7 ? 0 : KT - a.K;  // a shorter filter's taps are the window's last
  double taps[KT ? KT : 1];
#pragma unroll
  for (int i = 0; i < KT; ++i)
    taps[i] = i >= skip ? (double)a.taps[(a.taps_rows > 1 ? (int64_t)h * a.K : 0) + i - skip] : 0.0;
  // Group 0 has two blocks.  Groups of several waves meet at barriers, so there the others take a second, empty round.
  const int from = j == 0 ? 0 : j + 1, rounds = j == 0 || a.group > 64 ? 2 : 1;
  for (int r = 0; r < rounds; ++r) {
    const int i = from + r;
    const int64_t pos0 = (s & ~(int64_t)(BLOCK - 1)) + (int64_t)i * BLOCK;
    const int t0 = (int)max((int64_t)0, s - pos0);
    const int64_t left = s + n - pos0;
    const int t1 = (int)min((int64_t)BLOCK, left);
    bool live = fits && t1 > t0 && (r == 0 || j == 0);
    int64_t block = -1;
    if (live) block = c.block_at(b, h, pos0);
    live = live && block >= 0;
    double x[BLOCK];
    float y[BLOCK];
    double top_k = 0, top_v = 0;
    if (live && mine) {
      double w[HIST + BLOCK];
#pragma unroll
      for (int t = 0; t < HIST + BLOCK; ++t) {
        const int64_t at = pos0 - HIST + t - s;  // of the call's tokens
        w[t] = (double)to_f32(k[min(max(at, (int64_t)0), (int64_t)n - 1) * a.ksn]);
      }
      if (HIST && pos0 - HIST < s) {
#pragma unroll
        for (int t = 0; t < HIST + BLOCK - 1; ++t) {
          const int64_t pos = pos0 - HIST + t;
          if (pos < s) w[t] = pos >= 0 && s - pos < a.K ? (double)to_f32(raw[(pos & (RAW - 1)) * c.d]) : 0.0;
        }
      }
#pragma unroll
      for (int t = 0; t < BLOCK; ++t) {
        double acc = KT ? 0.0 : w[t];
#pragma unroll
        for (int u = 0; u < KT; ++u)
          if (KT == 7 || u >= skip) acc = fma(taps[u], w[t + u], acc);
        x[t] = acc;
        y[t] = to_f32(v[min(max(pos0 + t - s, (int64_t)0), (int64_t)n - 1) * a.vsn]);
        if (t >= t0 && t < t1) {
          if (fabs(acc) < __builtin_inf()) top_k = fmax(top_k, fabs(acc));
          if (fabsf(y[t]) < __builtin_inff()) top_v = fmax(top_v, (double)fabsf(y[t]));
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < BLOCK; ++t) x[t] = 0, y[t] = 0;
    }
    int ek = group_max(need(top_k), a.group, lds), ev = group_max(need(top_v), a.group, lds);
    if (!live) continue;
    const int was_k = min((int)c.k_scale[block], 247) - 127, was_v = min((int)c.v_scale[block], 247) - 127;
    if (t0 > 0) ek = max(ek, was_k), ev = max(ev, was_v);
    if (col >= c.D) continue;
    const double ik = __builtin_bit_cast(double, (uint64_t)(1023 - ek) << 52);
    const float iv = two_to(-ev);
    uint8_t* kb = c.k + block * BLOCK * c.D + col;
    uint8_t* vb = c.v + block * BLOCK * c.D + col * BLOCK;
    uint4 old = {0, 0, 0, 0};
    const bool part = t0 > 0 || t1 < BLOCK;
    if (part) old = *reinterpret_cast<const uint4*>(vb);
    const float again_k = ldexpf(1.0f, was_k - ek), again_v = ldexpf(1.0f, was_v - ev);
    unsigned out[4] = {0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < BLOCK; ++t) {
      unsigned byte;
      if (t < t0) {
        if (ek != was_k) kb[t * c.D] = (uint8_t)e4m3(value(kb[t * c.D]) * again_k);
        byte = e4m3(value(byte_of(old, t)) * again_v);
      } else if (t < t1) {
        const bool fk = fabs(x[t]) < __builtin_inf(), fv = fabsf(y[t]) < __builtin_inff();
        kb[t * c.D] = fk ? (uint8_t)e4m3(cut(x[t] * ik)) : E4M3_NAN;
        byte = fv ? e4m3(y[t] * iv) : E4M3_NAN;
      } else {
        byte = byte_of(old, t);
      }
      out[t >> 2] |= byte << (8 * (t & 3));
    }
    *reinterpret_cast<uint4*>(vb) = uint4{out[0], out[1], out[2], out[3]};
    if (col == 0) c.k_scale[block] = (uint8_t)(ek + 127), c.v_scale[block] = (uint8_t)(ev + 127);
  }
  if (c.raw && j == 0 && fits && mine)
    for (int t = max(0, n - RAW); t < n; ++t) raw[((s + t) & (RAW - 1)) * c.d] = k[t * a.ksn];
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
  const int64_t item = (int64_t)blockIdx.x * per + threadIdx.x / a.group;
  const int col = threadIdx.x & (a.group - 1);
  if (item >= a.items || col >= c.D) return;
  const int64_t bh = item / a.groups;
  const int b = (int)(bh / c.H), h = (int)(bh % c.H);
  const int64_t first = a.first ? a.first[b] : a.first_all;
  const int64_t pos0 = (first & ~(int64_t)(BLOCK - 1)) + item % a.groups * BLOCK;
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

template <typename T>
void append_any(const AppendArgs& a, int64_t grid, hipStream_t st) {
  const auto go = [&](auto kernel) { kernel<<<dim3((unsigned)grid), dim3(THREADS), 0, st>>>(a); };
  if (!a.taps) go(append_kernel<T, 0>);
  else if (a.K == 7) go(append_kernel<T, 7>);  // the framework's filters
  else go(append_kernel<T, 16>);
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
  a.group = group_of(a.c.D);
  const int64_t blocks = (N + 2 * BLOCK - 2) / BLOCK;  // a call may begin at a block's last token
  a.groups = (int)(blocks > 1 ? blocks - 1 : 1);
  a.items = (int64_t)a.c.B * a.c.H * a.groups;
  int64_t grid;
  if (int rc = grid_of(a.items, a.group, "cache_append", &grid)) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == PNFX_F32) append_any<float>(a, grid, st);
  else append_any<bf16>(a, grid, st);
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
