// One token of each row of logits: temperature, top-k, top-p and min-p from a given random number.
//
// With w_i = exp((z_i - max z) / temperature) and the tokens ordered by z, lower index first among equals, each of
// the three filters keeps the first so many, and what all keep is again the first so many: everything up to a
// threshold logit, and of the tokens that equal it those up to an index.  The token is the first by index at which
// the kept ones' running weight passes u times their whole weight.
//
// One workgroup of 16 waves has a row and goes over it several times, the next chunks on their way: the maximum; for
// top-k, the threshold by a histogram of max z - z, then of the logits' bits within its bin; for top-p, the same with the
// weights' sums; then the sum of each wave's 64 chunks, in the order of the row, the chunks in which u falls, and the
// token in them.
//
// bf16 rows have few different logits: with the magnitudes from 2^-32 to 2^16, 12289 of them.  Their weights are a table
// in LDS, one exponential for each that occurs, and one histogram of them settles both thresholds and the maximum: 256 rows of
// 131072 take 49 us (all weights one by one 150), of 1000 with top-p 15 (31), one of 33278 takes 19 (37); 64 rows of 4000
// by temperature alone 12 either way.
//
// Integers decide: weights are 64-bit fixed point, 2^S for the largest, so that sums are exact and the same in any
// order (the histogram's atomics among them).  S is 50, or 62 less the bits of V: 45 for 131072 tokens, 42 for 2^20.  The
// exponential is a table of 256 steps an octave times a cubic, in fp64 (1.4e-13, relative), and a weight is rounded by half
// a unit at most, so a border is off by no more than V 2^-(S+1) of the largest weight and 1.4e-13 of its own sum: 2^-29 of
// the largest in all for 131072 tokens, 2^-23 for 2^20, if every rounding falls to one side.  A token differs from the real
// numbers' only where u times the kept weight is as near to a border.  (An fp32 exponential moves some border past u every few
// hundred rows of 10^5 tokens.)
#include "pnfx_common.h"

#include <cmath>

namespace pnfx {
namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int DIGIT = 11, BINS = 1 << DIGIT;
constexpr float SPAN = 64;        // of the first histogram, at most: what lies further below shares its last bin
constexpr int MAX_PARTS = 257;    // chunks of a thread in the longest rows: 2^20 fp32, four a chunk, at any alignment
constexpr double LOG2E = 1.4426950408889634, LN2 = 0.6931471805599453;

struct SampleArgs {
  const void* z;
  int64_t rs;
  int V, S;  // S: bits behind the point of a weight
  const float* u;
  pnfx_sampling set;
  int64_t* tokens;
};

// Unsigned numbers in the order of the logits.
__device__ __forceinline__ unsigned key_of(float z) {
  const unsigned b = __builtin_bit_cast(unsigned, z);
  return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}

// A row, cut into 16-byte chunks, chunk c for thread c % THREADS: part j of all threads holds the logits right before
// part j + 1, and wave by wave in order.  Places beside the row hold -infinity, whose weight is 0.
template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T);  // elements of a chunk
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  const T* base;  // aligned: the row begins `off` elements behind it
  int off, V, parts;
  __device__ __forceinline__ Row(const T* p, int V_) : V(V_) {
    off = (int)(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
    base = p - off;
    parts = ((off + V + E - 1) / E + THREADS - 1) / THREADS;
  }
  __device__ __forceinline__ u32x4 read(int j) const {
    const int c = j * THREADS + threadIdx.x;
    if (c * E >= off && (c + 1) * E <= off + V) return *reinterpret_cast<const u32x4*>(base + c * E);
    u32x4 w = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int at = c * E + i - off;
      const float x = at >= 0 && at < V ? to_f32(base[c * E + i]) : -__builtin_inff();
      const unsigned bits = __builtin_bit_cast(unsigned, x);
      w[i * sizeof(T) / 4] |= sizeof(T) == 4 ? bits : i % 2 ? bits & 0xffff0000u : bits >> 16;
    }
    return w;
  }
  static __device__ __forceinline__ float element(const u32x4& w, int i) {  // -0 counts as 0
    const unsigned bits = sizeof(T) == 4 ? w[i] : i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16;
    return __builtin_bit_cast(float, bits) + 0.0f;
  }
  __device__ __forceinline__ int index(int j, int i) const { return (j * THREADS + (int)threadIdx.x) * E + i - off; }
  // f(part, its chunk), parts in order
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    constexpr int AHEAD = 2;
    u32x4 w[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (k < parts) w[k] = read(k);
    for (int j0 = 0; j0 < parts; j0 += AHEAD) {
      u32x4 next[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (j0 + AHEAD + k < parts) next[k] = read(j0 + AHEAD + k);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        if (j0 + k < parts) f(j0 + k, w[k]);
        w[k] = next[k];
      }
    }
  }
};

// Sums over a wave in registers: rows of 16 lanes, then from row to row (lanes without a source add 0).
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long moved(unsigned long long x) {
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)x, CTRL, ROWS, 0xf, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(x >> 32), CTRL, ROWS, 0xf, false);
  return (unsigned long long)hi << 32 | lo;
}
__device__ __forceinline__ unsigned long long wave_running(unsigned long long x) {
  x += moved<0x111, 0xf>(x);  // row_shr:1, 2, 4, 8
  x += moved<0x112, 0xf>(x);
  x += moved<0x114, 0xf>(x);
  x += moved<0x118, 0xf>(x);
  x += moved<0x142, 0xa>(x);  // row_bcast:15 into rows 1 and 3
  x += moved<0x143, 0xc>(x);  // row_bcast:31 into rows 2 and 3
  return x;
}
__device__ __forceinline__ unsigned long long lane_of(unsigned long long x, int lane) {
  return (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
         (unsigned)__builtin_amdgcn_readlane((int)(unsigned)x, lane);
}
__device__ __forceinline__ unsigned long long wave_total(unsigned long long x) { return lane_of(wave_running(x), 63); }

template <int STEPS>
struct Common {
  double table[STEPS];
  unsigned long long wave[WAVES];
  float top[WAVES], low[WAVES];
  unsigned long long before;
  int digit, found;
};
template <int STEPS>
struct Lds : Common<STEPS> {
  unsigned long long sums[MAX_PARTS * WAVES];  // of each part and wave; the histogram's bins
  unsigned count[BINS];
};
static_assert(BINS <= MAX_PARTS * WAVES, "");

// STEPS: of the table, an octave.  With 256 a cubic is 1.4e-13 off at most, relative, with 4096 a square 1.0e-13.
template <int STEPS>
struct Weights {
  const double* table;  // 2^S times the steps of an octave
  double c, top;        // steps of the table a unit of logit; the maximum
  double low;           // min_p's border, in steps
  float least;          // a logit of no weight in fixed point: about 2^-60 of the largest
  bool wide;            // there is none: the maximum is infinite, or temperatures are too low for fp32's steps there
  __device__ __forceinline__ void set(const double* t, float top_, double temperature, double min_p) {
    table = t, top = top_;
    c = fmin(STEPS * LOG2E / temperature, 1e300);
    low = min_p > 0 ? STEPS * log2(fmin(min_p, 1.0)) : -__builtin_inf();
    least = (float)fmax(top - 60.0 * STEPS / c, -3.4028234663852886e38);
    const double to = (least - top) * c;
    wide = !(to < -58.0 * STEPS && to > -61.0 * STEPS);
  }
  __device__ __forceinline__ double steps(float z) const {
    return wide && z == top ? 0.0 : ((double)z - top) * c;  // an infinite maximum: all others -infinity
  }
  __device__ __forceinline__ unsigned long long of_steps(double y) const {  // y >= -61 STEPS
    const double round = 6755399441055744.0;  // 1.5 * 2^52
    constexpr double A = LN2 / STEPS;
    const double t = y + round;
    const int n = (int)__builtin_bit_cast(uint64_t, t);
    const double r = y - (t - round);
    const double p = fma(r, STEPS == 256 ? fma(r, fma(r, A * A * A / 6, A * A / 2), A) : fma(r, A * A / 2, A), 1.0);
    constexpr int SHIFT = STEPS == 256 ? 8 : 12;
    const uint64_t e = (uint64_t)(uint32_t)(n >> SHIFT << 20) << 32;
    const double s = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, table[n & (STEPS - 1)]) + e);
    return __builtin_bit_cast(uint64_t, fma(s, p, 4503599627370496.0)) - 0x4330000000000000ull;  // the bits of 2^52
  }
  __device__ __forceinline__ unsigned long long operator()(float z) const {
    if (wide) return of_steps(fmax(steps(z), -60.0 * STEPS));
    return of_steps(((double)fmaxf(z, least) - top) * c);
  }
};

struct Cut {  // what is kept: logits of keys above, and those equal up to an index
  unsigned key;
  int index;
};

template <typename T, int STEPS>
struct Sampler {
  using R = Row<T>;
  using W = Weights<STEPS>;
  static constexpr int E = R::E;
  R row;
  Lds<STEPS>& s;
  int tid, lane, wave;
  float top, scale;  // the largest logit, and bins of the first histogram a unit below it
  __device__ __forceinline__ Sampler(const T* p, int V, Lds<STEPS>& lds) : row(p, V), s(lds) {
    tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  }
  __device__ __forceinline__ bool keeps(const Cut& cut, float z, int j, int i) const {
    const unsigned k = key_of(z);
    return k > cut.key || (k == cut.key && row.index(j, i) <= cut.index);
  }

  // First index at which the running sum of f(logit's bits, part, place) passes target(sum of all).
  template <typename F, typename G>
  __device__ __forceinline__ int first_of(unsigned long long* sums, F f, G target) const {
    const auto at_place = [&](const auto& w, int j, int i) {
      return f(sizeof(T) == 4 ? w[i] : w[i / 2] >> (i % 2 * 16), j, i);
    };
    __syncthreads();
    row.each([&](int j, const auto& w) {
      unsigned long long sum = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) sum += at_place(w, j, i);
      sum = __any(sum != 0) ? wave_total(sum) : 0;
      if (lane == 0) sums[j * WAVES + wave] = sum;
    });
    __syncthreads();
    // each wave finds the part and wave in which it is, 64 sums at a time
    unsigned long long all = 0, left = 0;
    const int n = row.parts * WAVES;
    for (int i = lane; i < n; i += 64) all += sums[i];
    left = target(wave_total(all));
    int at = n - 1;
    for (int i0 = 0; i0 < n; i0 += 64) {
      const unsigned long long mine = i0 + lane < n ? sums[i0 + lane] : 0, run = wave_running(mine);
      const unsigned long long hit = __ballot(run > left);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        at = i0 + l, left -= lane_of(run - mine, l);
        break;
      }
      left -= lane_of(run, 63);
    }
    if (wave == at % WAVES) {
      const int j = at / WAVES;
      const auto w = row.read(j);
      unsigned long long mine[E], sum = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) mine[i] = at_place(w, j, i), sum += mine[i];
      unsigned long long past = wave_running(sum) - sum;
      int found = -1;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (past <= left && left < past + mine[i]) found = row.index(j, i);
        past += mine[i];
      }
      const unsigned long long hit = __ballot(found >= 0);
      if (hit ? lane == __builtin_ctzll(hit) : lane == 0) s.found = found;
    }
    __syncthreads();
    return s.found;
  }
  // The same of the logits themselves.
  template <typename F, typename G>
  __device__ __forceinline__ int first(F f, G target) const {
    return first_of(
        s.sums,
        [&](unsigned bits, int j, int i) -> unsigned long long {
          const unsigned b = sizeof(T) == 4 ? bits : bits << 16;
          return f(__builtin_bit_cast(float, b) + 0.0f, j, i);
        },
        target);
  }

  __device__ __forceinline__ int bin(float z) const { return (int)fminf((top - z) * scale, (float)(BINS - 1)); }

  // The bin of s.sums (MASS) or s.count in which the target falls, from the last (down) or the first one on; what is
  // before it is taken off the target.
  template <bool MASS>
  __device__ __forceinline__ int fall(unsigned long long& target, bool down) const {
    const int bin = down ? BINS - 1 - 2 * tid : 2 * tid, next = down ? bin - 1 : bin + 1;
    const unsigned long long v0 = MASS ? s.sums[bin] : s.count[bin], v1 = MASS ? s.sums[next] : s.count[next];
    const unsigned long long run = wave_running(v0 + v1);
    if (lane == 63) s.wave[wave] = run;
    __syncthreads();
    unsigned long long past = run - v0 - v1;
    for (int w = 0; w < wave; ++w) past += s.wave[w];
    if (past < target && target <= past + v0) s.digit = bin, s.before = past;
    past += v0;
    if (past < target && target <= past + v1) s.digit = next, s.before = past;
    __syncthreads();
    target -= s.before;
    return s.digit;
  }
  __device__ __forceinline__ void clear() const {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BINS / THREADS; ++i) s.count[i * THREADS + tid] = 0, s.sums[i * THREADS + tid] = 0;
    __syncthreads();
  }

  // The threshold of the first tokens, in order, that have `target` (at least 1, at most all) in sum: of the kept
  // ones' weights, or of the kept ones themselves.
  template <bool MASS, typename G>
  __device__ __forceinline__ Cut threshold(const Cut& kept, const W& weight, G target_of) const {
    clear();
    row.each([&](int j, const auto& w) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float z = R::element(w, i);
        if (!keeps(kept, z, j, i)) continue;
        if (MASS) atomicAdd(&s.sums[bin(z)], weight(z));
        else atomicAdd(&s.count[bin(z)], 1u);
      }
    });
    __syncthreads();
    unsigned long long all = 0;
    for (int i = lane; i < BINS; i += 64) all += MASS ? s.sums[i] : s.count[i];
    unsigned long long target = target_of(wave_total(all));
    const int in = fall<MASS>(target, false);
    // Keys of the bin's logits: (top - z) scale is in [in, in + 1) but for roundings of 2^-24 each
    const double wide = 1.0 / scale;
    unsigned lo = 0, hi = key_of((float)((double)top - in * wide * (1 - 0x1p-20))) + 1;
    if (in < BINS - 1) lo = key_of((float)((double)top - (in + 1) * wide * (1 + 0x1p-20))) - 1;
    hi = max(min(hi, key_of(top)), lo);
    for (;;) {
      const int shift = max(0, 32 - __builtin_clz((hi - lo) | 1) - DIGIT);
      clear();
      row.each([&](int j, const auto& w) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float z = R::element(w, i);
          const unsigned d = key_of(z) - lo;
          if (d > hi - lo || bin(z) != in || !keeps(kept, z, j, i)) continue;
          atomicAdd(&s.count[d >> shift], 1u);
          if (MASS) atomicAdd(&s.sums[d >> shift], weight(z));
        }
      });
      __syncthreads();
      const int d = fall<MASS>(target, true);
      lo += (unsigned)d << shift, hi = lo + ((1u << shift) - 1);
      if (shift) continue;
      // equal tokens: how many of them
      const unsigned n = s.count[d];
      unsigned long long take = target;
      if (MASS) {
        const unsigned long long each = s.sums[d] / n;
        take = (target + each - 1) / each;
      }
      Cut cut{lo, row.V};
      if (take < n)
        cut.index = first([&](float z, int, int) -> unsigned long long { return key_of(z) == lo; },
                          [&](unsigned long long) { return take - 1; });
      if (kept.key == lo) cut.index = min(cut.index, kept.index);
      return cut;
    }
  }
};

// The table of bf16 rows: place 6144 for zero, those above it for the positive numbers from 2^-32 to 2^16, those
// below for the negative ones; what is beyond -2^16 shares the first, as its weight is 0.
constexpr int TINY = (127 - 32) << 7, HALF = 48 << 7, PLACES = 2 * HALF + 1;  // TINY: the bits of 2^-32
constexpr int MINE = 2 * HALF / THREADS;  // places of a thread; place 0 is nobody's, and nothing is counted there
constexpr int COPIES = 3;                 // of the histogram, for every third lane: neighbours meet in it often
struct Table {
  union {
    unsigned long long weight[PLACES];
    unsigned more[COPIES - 1][PLACES];
  };
  union {
    unsigned count[PLACES];
    struct {
      unsigned long long sums[(MAX_PARTS + 1) / 2 * WAVES];
      int ties[(MAX_PARTS + 1) / 2 * WAVES];
    };
  };
};
__device__ __forceinline__ int place_of(unsigned bits) {  // of bf16 bits
  const int d = min(max((int)(bits & 0x7fff), TINY - 1), TINY - 1 + HALF) - (TINY - 1);
  return HALF + (bits & 0x8000 ? -d : d);
}
__device__ __forceinline__ float number_at(int place) {
  const int d = place - HALF, b = d ? TINY - 1 + abs(d) : 0;
  return __builtin_bit_cast(float, (unsigned)(b | (d < 0 ? 0x8000 : 0)) << 16);
}

struct Settings {
  double top_p, u;
  int64_t top_k;
};

// A row whose logits the table holds: nothing between 0 and 2^-32, the largest below 2^16, no weight at -2^16.
struct FromTable {
  const Sampler<bf16, 256>& me;
  Table& t;
  const Weights<256>& w;
  int last, take;  // the last place that is kept, and how many of its tokens, the first ones

  // Counts the row's logits by places; the largest logit, or -infinity if the table does not hold the row.
  static __device__ __forceinline__ float histogram(const Sampler<bf16, 256>& me, Table& t) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    const int tid = me.tid;
    unsigned* const copy = tid % COPIES ? t.more[tid % COPIES - 1] : t.count;
    for (int i = tid; i < PLACES; i += THREADS) {
      t.count[i] = 0;
#pragma unroll
      for (int c = 0; c < COPIES - 1; ++c) t.more[c][i] = 0;
    }
    __syncthreads();
    u16x2 least = 0xffff, most = 0;  // magnitudes: the least but zero, less one; the largest
    me.row.each([&](int, const auto& x) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned pair = x[i];
        const u16x2 a = __builtin_bit_cast(u16x2, pair & 0x7fff7fffu);
        least = __builtin_elementwise_min(least, (u16x2)(a - (unsigned short)1));
        most = __builtin_elementwise_max(most, a);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int p = place_of(x[i / 2] >> (i % 2 * 16));
        if (p) atomicAdd(&copy[p], 1u);
      }
    });
    __syncthreads();
    unsigned sum[MINE];
    int top = 0;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int p = 1 + i * THREADS + tid;
      sum[i] = t.count[p];
#pragma unroll
      for (int c = 0; c < COPIES - 1; ++c) sum[i] += t.more[c][p];
      if (sum[i]) top = p;
    }
    if (min(least.x, least.y) < TINY - 1 || max(most.x, most.y) > 0x7f80) top = PLACES;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = max(top, __shfl_xor(top, o, 64));
    if (me.lane == 0) me.s.top[me.wave] = (float)top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MINE; ++i) t.count[1 + i * THREADS + tid] = sum[i];
    for (int i = 0; i < WAVES; ++i) top = max(top, (int)me.s.top[i]);
    return top == 0 || top >= PLACES - 1 ? -__builtin_inff() : number_at(top);
  }
  __device__ __forceinline__ void weights() const {  // of those that were counted
    for (int i = 0; i < MINE; ++i) {
      const int p = 1 + i * THREADS + me.tid;
      if (t.count[p]) t.weight[p] = w(number_at(p));
    }
    __syncthreads();
  }
  __device__ __forceinline__ void all_weights() const {
    for (int p = 1 + me.tid; p < PLACES; p += THREADS) {
      const float z = number_at(p);
      if (z <= me.top) t.weight[p] = w(z);
    }
  }

  // The place in which the target falls, going down by f(place, its tokens), and what of the target is left there.
  template <typename F, typename G>
  __device__ __forceinline__ int fall(F f, G target_of, unsigned long long* left) const {
    Lds<256>& s = me.s;
    const int p0 = PLACES - 1 - me.tid * MINE;
    unsigned long long v[MINE], sum = 0;
#pragma unroll
    for (int i = 0; i < MINE; ++i) v[i] = f(p0 - i, t.count[p0 - i]), sum += v[i];
    const unsigned long long run = wave_running(sum);
    if (me.lane == 63) s.wave[me.wave] = run;
    if (me.tid == 0) s.digit = 0, s.before = ~0ull;  // beyond all that is counted: nothing is cut
    __syncthreads();
    unsigned long long past = run - sum, all = 0;
    for (int i = 0; i < WAVES; ++i) past += i < me.wave ? s.wave[i] : 0, all += s.wave[i];
    const unsigned long long target = target_of(all);
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      if (past < target && target <= past + v[i]) s.digit = p0 - i, s.before = target - past;
      past += v[i];
    }
    __syncthreads();
    const int digit = s.digit;
    *left = s.before;
    __syncthreads();
    return digit;
  }

  // The first token at which the kept ones' running weight passes u times their whole weight.
  __device__ __forceinline__ int token(double u, bool ties) const {
    Lds<256>& s = me.s;
    const int lane = me.lane, wave = me.wave;
    const unsigned long long tie = last > 0 ? t.weight[last] : 0;
    __syncthreads();
    me.row.each([&](int j, const auto& x) {
      unsigned long long sum = 0;
      int equal = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int p = place_of(x[i / 2] >> (i % 2 * 16));
        if (p > last) sum += t.weight[p];
        if (ties) equal += __popcll(__ballot(p == last));
      }
      sum = __any(sum != 0) ? wave_total(sum) : 0;
      if (lane == 0) t.sums[j * WAVES + wave] = sum, t.ties[j * WAVES + wave] = equal;
    });
    __syncthreads();
    const int n = me.row.parts * WAVES;
    // `before`: the equal ones in what lies before; of a sum's own, so many as are still kept count
    const auto whole = [&](int i, unsigned long long& before) {
      unsigned long long sum = i < n ? t.sums[i] : 0;
      if (ties) {
        const int mine = i < n ? t.ties[i] : 0;
        const unsigned long long run = wave_running((unsigned long long)mine);
        sum += tie * (unsigned)min(mine, max(0, take - (int)(before + run) + mine));
        before += lane_of(run, 63);
      }
      return sum;
    };
    unsigned long long all = 0, before = 0;
    for (int i0 = 0; i0 < n; i0 += 64) all += whole(i0 + lane, before);
    all = wave_total(all);
    unsigned long long left = min((unsigned long long)(u * (double)all), all - 1);
    before = 0;
    int at = n - 1, equal = 0;
    for (int i0 = 0; i0 < n; i0 += 64) {
      const unsigned long long was = before, mine = whole(i0 + lane, before), run = wave_running(mine);
      const unsigned long long hit = __ballot(run > left);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        at = i0 + l, left -= lane_of(run - mine, l);
        if (ties) {
          const unsigned long long c = lane < l ? t.ties[i0 + lane] : 0;
          equal = (int)(was + wave_total(c));
        }
        break;
      }
      left -= lane_of(run, 63);
    }
    if (wave == at % WAVES) {
      const int j = at / WAVES;
      const auto x = me.row.read(j);
      int p[8], mine = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = place_of(x[i / 2] >> (i % 2 * 16)), mine += p[i] == last;
      equal += (int)wave_running((unsigned long long)mine) - mine;
      unsigned long long v[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = p[i] > last ? t.weight[p[i]] : ties && p[i] == last && equal < take ? tie : 0;
        equal += p[i] == last;
        sum += v[i];
      }
      unsigned long long past = wave_running(sum) - sum;
      int found = -1;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (past <= left && left < past + v[i]) found = me.row.index(j, i);
        past += v[i];
      }
      const unsigned long long hit = __ballot(found >= 0);
      if (hit ? lane == __builtin_ctzll(hit) : lane == 0) s.found = found;
    }
    __syncthreads();
    return s.found;
  }

  __device__ __forceinline__ int run(const Settings& set) {
    const bool by_k = set.top_k > 0 && set.top_k < me.row.V, by_p = set.top_p < 1;
    last = 0, take = 0;
    bool ties = false;
    if (by_k || by_p) {
      weights();
      unsigned long long left;
      if (by_k) {
        last = fall([](int, unsigned c) -> unsigned long long { return c; },
                    [&](unsigned long long) { return (unsigned long long)set.top_k; }, &left);
        take = (int)min(left, (unsigned long long)(1 << 30));
      }
      if (by_p) {
        const auto kept = [&](int p, unsigned c) { return p > last ? c : p == last && by_k ? min(c, (unsigned)take) : !by_k ? c : 0; };
        const int to = fall([&](int p, unsigned c) { return c ? t.weight[p] * kept(p, c) : 0; },
                            [&](unsigned long long all) {
                              const double part = ceil(fmax(set.top_p, 0.0) * (double)all);
                              return min(max((unsigned long long)part, 1ull), all);
                            }, &left);
        const unsigned long long each = t.weight[to], most = kept(to, t.count[to]);
        take = (int)min((left + each - 1) / each, most), last = to;
      }
      ties = last > 0 && (unsigned)take < t.count[last];
      if (last > 0 && !ties) last -= 1;  // all of its tokens: what is above the place below it
    } else {
      all_weights();
    }
    if (w.low > -__builtin_inf()) {  // the last place that min_p drops
      int lo = 0, hi = PLACES - 1;
      while (hi > lo) {
        const int mid = (lo + hi + 1) / 2;
        if (w.steps(number_at(mid)) < w.low) lo = mid;
        else hi = mid - 1;
      }
      if (lo > last || (lo == last && ties)) last = lo, ties = false;
    }
    return token(set.u, ties);
  }
};

template <bool TABLE>
union Shared {
  Lds<4096> s;
  __device__ Shared() {}
};
template <>
union Shared<true> {
  Lds<256> s;
  struct {
    Common<256> common;
    Table table;
  } t;
  __device__ Shared() {}
};

template <typename T, bool TABLE>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleArgs a) {
  __shared__ Shared<TABLE> shared;
  constexpr int STEPS = TABLE ? 256 : 4096;
  Lds<STEPS>& s = shared.s;
  const int64_t b = blockIdx.x;
  const pnfx_sampling& set = a.set;
  const double temperature = set.temperature_each ? (double)set.temperature_each[b] : set.temperature;
  const int64_t top_k = set.top_k_each ? (int64_t)set.top_k_each[b] : set.top_k;
  const double top_p = set.top_p_each ? (double)set.top_p_each[b] : set.top_p;
  const double min_p = set.min_p_each ? (double)set.min_p_each[b] : set.min_p;
  const double u = fmin(fmax((double)a.u[b], 0.0), 1.0);
  Sampler<T, STEPS> me(static_cast<const T*>(a.z) + b * a.rs, a.V, s);
  using R = Row<T>;
  const bool cut_off = (top_k > 0 && top_k < a.V) || top_p < 1;
  if (me.tid < 256) s.table[STEPS / 256 * me.tid] = ldexp(exp2(me.tid * (1.0 / 256)), a.S);
  const Settings settings{top_p, u, top_k};
  bool counted = false;
  if constexpr (TABLE) {
    counted = cut_off && temperature > 0 && top_k != 1;
    if (counted) {  // the maximum comes from the counts, with one reading of the row less
      me.top = FromTable::histogram(me, shared.t.table);
      Weights<STEPS> w;
      w.set(s.table, me.top, temperature, min_p);
      if (me.top > -__builtin_inff() && !w.wide && w.least > -65280.0f) {
        const int token = FromTable{me, shared.t.table, w, 0, 0}.run(settings);
        if (me.tid == 0) a.tokens[b] = token;
        return;
      }
      __syncthreads();  // s.top
    }
  }
  float top = -__builtin_inff(), low = __builtin_inff(), tiny = __builtin_inff();
  me.row.each([&](int, const auto& w) {
#pragma unroll
    for (int i = 0; i < R::E; ++i) {
      const float z = R::element(w, i);
      top = __builtin_elementwise_maximum(top, z);  // a NaN stays
      if (!TABLE) low = fminf(low, fabsf(z) < __builtin_inff() ? z : low);
      else tiny = fminf(tiny, z != 0 ? fabsf(z) : tiny);
    }
  });
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    top = __builtin_elementwise_maximum(top, __shfl_xor(top, o, 64));
    low = fminf(low, __shfl_xor(low, o, 64));
    if (TABLE) tiny = fminf(tiny, __shfl_xor(tiny, o, 64));
  }
  if (!TABLE) {  // the steps between
    __syncthreads();
    double between = 1, step = 1 + LN2 / STEPS + LN2 / STEPS * (LN2 / STEPS) / 2 + LN2 / STEPS * (LN2 / STEPS) * (LN2 / STEPS) / 6;
    const int part = me.tid & 255, from = me.tid >> 8;
    for (int i = 1; i < STEPS / 256; ++i) {
      between *= step;
      if (i % 4 == from) s.table[STEPS / 256 * part + i] = s.table[STEPS / 256 * part] * between;
    }
  }
  if (me.lane == 0) s.top[me.wave] = top, s.low[me.wave] = TABLE ? tiny : low;
  __syncthreads();
  for (int w = 0; w < WAVES; ++w) {
    top = __builtin_elementwise_maximum(top, s.top[w]);
    if (TABLE) tiny = fminf(tiny, s.low[w]);
    else low = fminf(low, s.low[w]);
  }
  int token = -1;
  if (top > -__builtin_inff()) {  // neither NaN nor nothing
    if (!(temperature > 0) || top_k == 1) {
      token = me.first([&](float z, int, int) -> unsigned long long { return z == top; },
                       [](unsigned long long) { return 0ull; });
    } else {
      Weights<STEPS> w;
      w.set(s.table, top, temperature, min_p);
      me.top = top;
      if constexpr (TABLE) {
        if (!counted && tiny >= 0x1p-32f && top < 65536.0f && !w.wide && w.least > -65280.0f) {
          token = FromTable{me, shared.t.table, w, 0, 0}.run(settings);
          if (me.tid == 0) a.tokens[b] = token;
          return;
        }
        low = top - SPAN;
      }
      // of an infinite maximum, the finite logits are all in the last bin
      me.scale = top == __builtin_inff() ? 1.0f : (BINS - 1) / fmaxf(fminf(top - low, SPAN), 1e-30f);
      Cut cut{0, a.V};
      if (top_k > 0 && top_k < a.V)
        cut = me.template threshold<false>(cut, w, [&](unsigned long long) { return (unsigned long long)top_k; });
      if (top_p < 1)
        cut = me.template threshold<true>(cut, w, [&](unsigned long long all) {
          const double part = ceil(fmax(top_p, 0.0) * (double)all);
          return min(max((unsigned long long)part, 1ull), all);
        });
      const auto target = [&](unsigned long long all) { return min((unsigned long long)(u * (double)all), all - 1); };
      if (cut.key == 0 && !(min_p > 0))
        token = me.first([&](float z, int, int) { return w(z); }, target);
      else
        token = me.first(
            [&](float z, int j, int i) -> unsigned long long {
              return me.keeps(cut, z, j, i) && w.steps(z) >= w.low ? w(z) : 0;
            },
            target);
    }
  }
  if (me.tid == 0) a.tokens[b] = token;
}

template <typename T>
void sample_any(const SampleArgs& a, int64_t B, hipStream_t st) {
  const dim3 grid((unsigned)B), block(THREADS);
  sample_kernel<T, sizeof(T) == 2><<<grid, block, 0, st>>>(a);
}

}  // namespace
}  // namespace pnfx

extern "C" int pnfx_sample(const void* logits, int64_t rs, int64_t B, int64_t V, const float* u,
                           const pnfx_sampling* settings, int64_t* tokens, int dtype, void* stream) {
  using namespace pnfx;
  PNFX_REQUIRE(logits && u && settings && tokens, "sample: null pointer");
  PNFX_REQUIRE(dtype == PNFX_F32 || dtype == PNFX_BF16, "sample: dtype %d", dtype);
  PNFX_REQUIRE(B >= 1 && B < (1 << 22) && V >= 1 && V <= (1 << 20), "sample: B=%lld V=%lld", (long long)B, (long long)V);
  PNFX_REQUIRE(rs >= V || B == 1, "sample: row stride %lld", (long long)rs);
  int bits = 0;
  while ((1ll << bits) < V) ++bits;
  const SampleArgs a{logits, rs, (int)V, std::min(50, 62 - bits), u, *settings, tokens};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == PNFX_F32) sample_any<float>(a, B, st);
  else sample_any<bf16>(a, B, st);
  return launch_status("sample");
}
