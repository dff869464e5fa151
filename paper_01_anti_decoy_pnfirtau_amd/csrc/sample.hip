// One token of each row of logits: temperature, top-k, top-p and min-p from a given random number.
//
// With w_i = exp((z_i - max z) / temperature) and the tokens ordered by z, lower index first among equals, each of
// the three filters keeps the first so many, and what all keep is again the first so many: everything up to a
// threshold logit, and of the tokens that equal it those up to an index.  The token is the first by index at which
// the kept ones' running weight passes u times their whole weight.
//
// One workgroup of 16 waves has a row, in registers where it fits them, and goes over it several times: the maximum;
// for top-k, the threshold by a histogram of max z - z, then of the logits' bits within its bin; for top-p, the same
// with the weights' sums; then the sum of each wave's 64 chunks, in the order of the row, the chunks in which u falls,
// and the token in them.
//
// Integers decide: weights are 64-bit fixed point, 2^S for the largest, so that sums are exact and the same in any
// order (the histogram's atomics among them), and a token differs from the real numbers' only where u falls within about
// 2^-46 of a border.  For that the exponential is a table of 256 steps an octave times a cubic, in fp64 (1.4e-13,
// relative): one of fp32 is off by enough to move some border past u every few hundred rows of 10^5 tokens.
#include "pnfx_common.h"

#include <cmath>

namespace pnfx {
namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int DIGIT = 11, BINS = 1 << DIGIT;
constexpr int STEPS = 256;        // of the exponential's table, an octave
constexpr float SPAN = 64;        // of the first histogram, at most: what lies further below shares its last bin
constexpr int MAX_PARTS = 256;    // chunks of a thread in the longest rows: 2^20 fp32, four a chunk
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
// part j + 1, and wave by wave in order.  PARTS: those that a thread has in registers, 0: read again each time.  Places
// beside the row hold -infinity, whose weight is 0.
template <typename T, int PARTS>
struct Row {
  static constexpr int E = 16 / sizeof(T);  // elements of a chunk
  static constexpr int KEEP = PARTS ? PARTS : 1;
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  const T* base;  // aligned: the row begins `off` elements behind it
  int off, V, chunks, parts;
  u32x4 kept[KEEP];
  __device__ __forceinline__ Row(const T* p, int V_) : V(V_) {
    off = (int)(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
    base = p - off;
    chunks = (off + V + E - 1) / E;
    parts = PARTS ? PARTS : (chunks + THREADS - 1) / THREADS;
#pragma unroll
    for (int j = 0; j < PARTS; ++j) kept[j] = read(j);
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
    if (PARTS) {
#pragma unroll
      for (int j = 0; j < PARTS; ++j) {
        u32x4 w = kept[j];
        asm volatile("" : "+v"(w));  // what a pass makes of the chunks is not held for the next one
        f(j, w);
      }
    } else {
      constexpr int AHEAD = 4;
      for (int j0 = 0; j0 < parts; j0 += AHEAD) {
        u32x4 w[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
          if (j0 + k < parts) w[k] = read(j0 + k);
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
          if (j0 + k < parts) f(j0 + k, w[k]);
      }
    }
  }
  __device__ __forceinline__ u32x4 part(int j) const {
    if (!PARTS) return read(j);
    u32x4 w = kept[0];
#pragma unroll
    for (int k = 1; k < PARTS; ++k)
      if (k == j) w = kept[k];
    return w;
  }
};

struct Lds {
  double table[STEPS];
  unsigned long long sums[MAX_PARTS * WAVES];  // of each part and wave; the histogram's bins
  unsigned count[BINS];
  unsigned long long wave[WAVES];
  float top[WAVES], low[WAVES];
  unsigned long long before;
  int digit, found;
};
static_assert(BINS <= MAX_PARTS * WAVES, "");

struct Weights {
  const double* table;  // 2^S times the steps of an octave
  double c, top;        // steps of the table a unit of logit; the maximum
  double low;           // min_p's border, in steps
  bool infinite;        // the maximum is: it alone has a weight
  __device__ __forceinline__ double steps(float z) const {
    if (infinite) return z == __builtin_inff() ? 0.0 : -__builtin_inf();
    return ((double)z - top) * c;
  }
  __device__ __forceinline__ unsigned long long of_steps(double y) const {
    const double round = 6755399441055744.0;  // 1.5 * 2^52
    constexpr double A = LN2 / STEPS;
    y = fmax(y, -60.0 * STEPS);  // 2^-60: 0 in fixed point
    const double t = y + round;
    const int n = (int)__builtin_bit_cast(uint64_t, t);
    const double r = y - (t - round);
    const double p = fma(r, fma(r, fma(r, A * A * A / 6, A * A / 2), A), 1.0);
    const uint64_t s = __builtin_bit_cast(uint64_t, table[n & (STEPS - 1)]) + ((uint64_t)(uint32_t)(n >> 8 << 20) << 32);
    return __builtin_bit_cast(uint64_t, fma(__builtin_bit_cast(double, s), p, 4503599627370496.0)) -
           0x4330000000000000ull;  // the bits of 2^52
  }
  __device__ __forceinline__ unsigned long long operator()(float z) const { return of_steps(steps(z)); }
};

__device__ __forceinline__ unsigned long long wave_total(unsigned long long x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}
__device__ __forceinline__ unsigned long long wave_running(unsigned long long x, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const unsigned long long y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  return x;
}

struct Cut {  // what is kept: logits of keys above, and those equal up to an index
  unsigned key;
  int index;
};

template <typename T, int PARTS>
struct Sampler {
  using R = Row<T, PARTS>;
  static constexpr int E = R::E;
  R row;
  Lds& s;
  int tid, lane, wave;
  float top, scale;  // the largest logit, and bins of the first histogram a unit below it
  __device__ __forceinline__ Sampler(const T* p, int V, Lds& lds) : row(p, V), s(lds) {
    tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  }
  __device__ __forceinline__ bool keeps(const Cut& cut, float z, int j, int i) const {
    const unsigned k = key_of(z);
    return k > cut.key || (k == cut.key && row.index(j, i) <= cut.index);
  }

  // First index at which the running sum of f(logit, part, place) passes target(sum of all).
  template <typename F, typename G>
  __device__ __forceinline__ int first(F f, G target) const {
    __syncthreads();
    row.each([&](int j, const auto& w) {
      unsigned long long sum = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) sum += f(R::element(w, i), j, i);
      sum = __any(sum != 0) ? wave_total(sum) : 0;
      if (lane == 0) s.sums[j * WAVES + wave] = sum;
    });
    __syncthreads();
    // each wave finds the part and wave in which it is, 64 sums at a time
    unsigned long long all = 0, left = 0;
    const int n = row.parts * WAVES;
    for (int i = lane; i < n; i += 64) all += s.sums[i];
    left = target(wave_total(all));
    int at = n - 1;
    for (int i0 = 0; i0 < n; i0 += 64) {
      const unsigned long long mine = i0 + lane < n ? s.sums[i0 + lane] : 0, run = wave_running(mine, lane);
      const unsigned long long hit = __ballot(run > left);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        at = i0 + l, left -= __shfl(run - mine, l, 64);
        break;
      }
      left -= __shfl(run, 63, 64);
    }
    if (wave == at % WAVES) {
      const int j = at / WAVES;
      const auto w = row.part(j);
      unsigned long long mine[E], sum = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) mine[i] = f(R::element(w, i), j, i), sum += mine[i];
      unsigned long long past = wave_running(sum, lane) - sum;
      int found = -1;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (past <= left && left < past + mine[i]) found = row.index(j, i);
        past += mine[i];
      }
      const unsigned long long hit = __ballot(found >= 0);
      if (lane == 0) s.found = -1;
      if (found >= 0 && lane == __builtin_ctzll(hit)) s.found = found;
    }
    __syncthreads();
    return s.found;
  }

  __device__ __forceinline__ int bin(float z) const { return (int)fminf((top - z) * scale, (float)(BINS - 1)); }

  // The bin of s.sums (MASS) or s.count in which the target falls, from the last (down) or the first one on; what is
  // before it is taken off the target.
  template <bool MASS>
  __device__ __forceinline__ int fall(unsigned long long& target, bool down) const {
    const int bin = down ? BINS - 1 - 2 * tid : 2 * tid, next = down ? bin - 1 : bin + 1;
    const unsigned long long v0 = MASS ? s.sums[bin] : s.count[bin], v1 = MASS ? s.sums[next] : s.count[next];
    const unsigned long long run = wave_running(v0 + v1, lane);
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
  __device__ __forceinline__ Cut threshold(const Cut& kept, const Weights& weight, G target_of) const {
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

template <typename T, int PARTS>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleArgs a) {
  __shared__ Lds s;
  const int64_t b = blockIdx.x;
  const pnfx_sampling& set = a.set;
  const double temperature = set.temperature_each ? (double)set.temperature_each[b] : set.temperature;
  const int64_t top_k = set.top_k_each ? (int64_t)set.top_k_each[b] : set.top_k;
  const double top_p = set.top_p_each ? (double)set.top_p_each[b] : set.top_p;
  const double min_p = set.min_p_each ? (double)set.min_p_each[b] : set.min_p;
  const double u = fmin(fmax((double)a.u[b], 0.0), 1.0);
  Sampler<T, PARTS> me(static_cast<const T*>(a.z) + b * a.rs, a.V, s);
  using R = Row<T, PARTS>;
  if (me.tid < STEPS) s.table[me.tid] = ldexp(exp2(me.tid * (1.0 / STEPS)), a.S);
  float top = -__builtin_inff(), low = __builtin_inff();
  me.row.each([&](int, const auto& w) {
#pragma unroll
    for (int i = 0; i < R::E; ++i) {
      const float z = R::element(w, i);
      top = __builtin_elementwise_maximum(top, z);  // a NaN stays
      low = fminf(low, fabsf(z) < __builtin_inff() ? z : low);
    }
  });
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    top = __builtin_elementwise_maximum(top, __shfl_xor(top, o, 64));
    low = fminf(low, __shfl_xor(low, o, 64));
  }
  if (me.lane == 0) s.top[me.wave] = top, s.low[me.wave] = low;
  __syncthreads();
  for (int w = 0; w < WAVES; ++w) top = __builtin_elementwise_maximum(top, s.top[w]), low = fminf(low, s.low[w]);
  int token = -1;
  if (top > -__builtin_inff()) {  // neither NaN nor nothing
    if (!(temperature > 0) || top_k == 1) {
      token = me.first([&](float z, int, int) -> unsigned long long { return z == top; },
                       [](unsigned long long) { return 0ull; });
    } else {
      Weights w;
      w.table = s.table, w.infinite = top == __builtin_inff();
      w.c = fmin(STEPS * LOG2E / temperature, 1e300), w.top = top;
      w.low = min_p > 0 ? STEPS * log2(fmin(min_p, 1.0)) : -__builtin_inf();
      // of an infinite maximum, the finite logits are all in the last bin
      me.top = top;
      me.scale = w.infinite ? 1.0f : (BINS - 1) / fmaxf(fminf(top - low, SPAN), 1e-30f);
      Cut cut{0, a.V};
      if (top_k > 0 && top_k < a.V)
        cut = me.template threshold<false>(cut, w, [&](unsigned long long) { return (unsigned long long)top_k; });
      if (top_p < 1)
        cut = me.template threshold<true>(cut, w, [&](unsigned long long all) {
          const double part = ceil(fmax(top_p, 0.0) * (double)all);
          return min(max((unsigned long long)part, 1ull), all);
        });
      token = me.first(
          [&](float z, int j, int i) -> unsigned long long {
            if (!me.keeps(cut, z, j, i)) return 0;
            const double y = w.steps(z);
            return y >= w.low ? w.of_steps(y) : 0;
          },
          [&](unsigned long long all) { return min((unsigned long long)(u * (double)all), all - 1); });
    }
  }
  if (me.tid == 0) a.tokens[b] = token;
}

template <typename T>
void sample_any(const SampleArgs& a, int64_t B, hipStream_t st) {
  const auto go = [&](auto kernel) { kernel<<<dim3((unsigned)B), dim3(THREADS), 0, st>>>(a); };
  const int parts = (a.V + 2 * (16 / (int)sizeof(T)) - 2) / (16 / (int)sizeof(T) * THREADS) + 1;  // at any alignment
  if (parts <= 2) go(sample_kernel<T, 2>);
  else if (parts <= 5) go(sample_kernel<T, 5>);
  else if (parts <= 9) go(sample_kernel<T, 9>);
  else go(sample_kernel<T, 0>);
}

}  // namespace
}  // namespace pnfx

extern "C" int pnfx_sample(const void* logits, int64_t rs, int64_t B, int64_t V, const float* u,
                           const pnfx_sampling* settings, int64_t* tokens, int dtype, void* stream) {
  using namespace pnfx;
  PNFX_REQUIRE(logits && u && settings && tokens, "sample: null pointer");
  PNFX_REQUIRE(dtype == PNFX_F32 || dtype == PNFX_BF16, "sample: dtype %d", dtype);
  PNFX_REQUIRE(B >= 1 && B < (1 << 22) && V >= 1 && V < (1 << 20), "sample: B=%lld V=%lld", (long long)B, (long long)V);
  PNFX_REQUIRE(rs >= V || B == 1, "sample: row stride %lld", (long long)rs);
  int bits = 0;
  while ((1ll << bits) < V) ++bits;
  const SampleArgs a{logits, rs, (int)V, std::min(50, 62 - bits), u, *settings, tokens};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == PNFX_F32) sample_any<float>(a, B, st);
  else sample_any<bf16>(a, B, st);
  return launch_status("sample");
}
