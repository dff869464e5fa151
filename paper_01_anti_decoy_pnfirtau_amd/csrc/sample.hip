// One token of each row of logits: temperature, top-k, top-p and min-p from a given random number.
//
// With w_i = exp((z_i - max z) / temperature) and the tokens ordered by z, lower index first among equals, each of
// the three filters keeps the first so many, and what all keep is again the first so many: everything up to a
// threshold logit, and of the tokens that equal it those up to an index.  The token is the first by index at which
// the kept ones' running weight passes u times their whole weight.
//
// One workgroup of 16 waves has a row and passes over it several times, from its L2 or the memory-side cache after
// the first: the maximum; for top-k, the threshold by a histogram of the logits' leading bits, then of the next ones
// within its bin; for top-p, the same with the weights' sums; then the waves' sums in order, the wave's part in which
// u falls, and so on down to the token.
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
constexpr int STEPS = 256;  // of the exponential's table, an octave
constexpr double LOG2E = 1.4426950408889634, LN2 = 0.6931471805599453;

struct SampleArgs {
  const void* z;
  int64_t rs;
  int V, S;  // S: bits behind the point of a weight
  const float* u;
  pnfx_sampling set;
  int64_t* tokens;
};

template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T);  // elements of a 16-byte chunk
  const T* base;  // aligned: the row begins `off` elements behind it
  int off, V, chunks;
  __device__ __forceinline__ Row(const T* p, int V_) : V(V_) {
    off = (int)(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
    base = p - off;
    chunks = (off + V + E - 1) / E;
  }
  __device__ __forceinline__ bool whole(int c) const { return c * E >= off && (c + 1) * E <= off + V; }
  // The chunk's elements; those beside the row are left.
  __device__ __forceinline__ void load(int c, float (&x)[E]) const {
    if (whole(c)) {
      const uint4 w = *reinterpret_cast<const uint4*>(base + c * E);
      T t[E];
      *reinterpret_cast<uint4*>(t) = w;
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = to_f32(t[i]);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int at = c * E + i - off;
        x[i] = at >= 0 && at < V ? to_f32(base[c * E + i]) : 0.0f;
      }
    }
  }
  // f(index, logit) for the elements of every step-th chunk from c0 on before c1; several loads on their way.
  template <typename F>
  __device__ __forceinline__ void each(int c0, int c1, int step, F f) const {
    constexpr int AHEAD = 4;
    for (int c = c0; c < c1; c += AHEAD * step) {
      float x[AHEAD][E];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (c + j * step < c1) load(c + j * step, x[j]);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (c + j * step < c1) {
          const int at = (c + j * step) * E - off;
#pragma unroll
          for (int i = 0; i < E; ++i)
            if ((unsigned)(at + i) < (unsigned)V) f(at + i, x[j][i] + 0.0f);  // -0 counts as 0
        }
    }
  }
};

// Unsigned numbers in the order of the logits; bf16 ones have their 16 bits.
template <typename T>
__device__ __forceinline__ unsigned key_of(float z) {
  const unsigned b = __builtin_bit_cast(unsigned, z);
  const unsigned k = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  return sizeof(T) == 2 ? k >> 16 : k;
}

struct Lds {
  double table[STEPS];
  unsigned count[BINS];
  unsigned long long mass[BINS];
  unsigned long long sums[WAVES];
  float top[WAVES];
  int flag[WAVES];
  unsigned long long before;
  int digit, index;
};

struct Weights {
  const double* table;
  float zmax;
  double c;    // steps of the table a unit of logit
  double low;  // min_p's border, in steps
  int S;
  __device__ __forceinline__ double steps(float z) const {
    return z == zmax ? 0.0 : ((double)z - (double)zmax) * c;  // an infinite maximum's other tokens: -infinity
  }
  __device__ __forceinline__ unsigned long long of_steps(double y) const {
    const double round = 6755399441055744.0;  // 1.5 * 2^52
    y = fmax(y, -60.0 * STEPS);               // 2^-60: 0 in fixed point
    const double t = y + round;
    const int n = (int)__builtin_bit_cast(uint64_t, t);
    const double r = (y - (t - round)) * (LN2 / STEPS);
    const double p = fma(r, fma(r, fma(r, 1.0 / 6, 0.5), 1.0), 1.0);
    const double s = table[n & (STEPS - 1)] * __builtin_bit_cast(double, (uint64_t)((n >> 8) + S + 1023) << 52);
    return __builtin_bit_cast(uint64_t, fma(s, p, 4503599627370496.0)) & 0xfffffffffffffull;  // + 2^52
  }
  __device__ __forceinline__ unsigned long long operator()(float z) const { return of_steps(steps(z)); }
};

__device__ __forceinline__ unsigned long long wave_total(unsigned long long x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}

struct Cut {  // what is kept: logits of keys above, and those equal up to an index
  unsigned key;
  int index;
  __device__ __forceinline__ bool keeps(unsigned k, int i) const { return k > key || (k == key && i <= index); }
};

template <typename T>
struct Sampler {
  Row<T> row;
  Lds& s;
  int tid, lane, wave;
  __device__ __forceinline__ Sampler(const T* p, int V, Lds& lds) : row(p, V), s(lds) {
    tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  }

  // First index at which the running sum of f(index, logit) passes target(sum of all).
  template <typename F, typename G>
  __device__ __forceinline__ int first(F f, G target) const {
    int c0 = 0, c1 = row.chunks;
    unsigned long long left = 0;
    for (bool whole = true;; whole = false) {
      const int per = (c1 - c0 + WAVES - 1) / WAVES;
      const int from = min(c0 + wave * per, c1), to = min(from + per, c1);
      unsigned long long sum = 0;
      row.each(from + lane, to, 64, [&](int i, float z) { sum += f(i, z); });
      sum = wave_total(sum);
      __syncthreads();
      if (lane == 0) s.sums[wave] = sum;
      __syncthreads();
      if (whole) {
        unsigned long long all = 0;
        for (int w = 0; w < WAVES; ++w) all += s.sums[w];
        left = target(all);
      }
      int w = 0;
      while (w < WAVES - 1 && left >= s.sums[w]) left -= s.sums[w++];
      c0 = min(c0 + w * per, c1), c1 = min(c0 + per, c1);
      if (c1 - c0 <= 64) break;
    }
    // one chunk a lane
    constexpr int E = Row<T>::E;
    float x[E];
    unsigned long long mine[E], sum = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) mine[i] = 0;
    const int c = c0 + lane;
    if (c < c1) {
      row.load(c, x);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int at = c * E + i - row.off;
        if ((unsigned)at < (unsigned)row.V) mine[i] = f(at, x[i] + 0.0f);
        sum += mine[i];
      }
    }
    unsigned long long run = sum;
    for (int o = 1; o < 64; o *= 2) {
      const unsigned long long y = __shfl_up(run, o, 64);
      if (lane >= o) run += y;
    }
    unsigned long long past = run - sum;
    int found = row.V;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (past <= left && left < past + mine[i]) found = c * E + i - row.off;
      past += mine[i];
    }
    const unsigned long long hit = __ballot(found < row.V);
    return hit ? __shfl(found, __builtin_ctzll(hit), 64) : row.V - 1;
  }

  // The threshold of the first tokens, in order, that have `target` (at least 1, at most all) in sum: of the kept
  // ones' weights, or of the kept ones themselves.
  template <bool MASS, typename G>
  __device__ __forceinline__ Cut threshold(const Cut& kept, const Weights& weight, G target_of) const {
    constexpr int BITS = sizeof(T) * 8;
    unsigned prefix = 0;
    unsigned long long target = 0;
    for (int level = 0, high = BITS;; ++level) {
      const int shift = max(high - DIGIT, 0), digits = high - shift;
      for (int i = tid; i < (1 << digits); i += THREADS) {
        s.count[i] = 0;
        if (MASS) s.mass[i] = 0;
      }
      __syncthreads();
      row.each(tid, row.chunks, THREADS, [&](int i, float z) {
        const unsigned k = key_of<T>(z);
        if ((level && k >> high != prefix) || !kept.keeps(k, i)) return;
        const unsigned d = (k >> shift) & ((1u << digits) - 1);
        atomicAdd(&s.count[d], 1u);
        if (MASS) atomicAdd(&s.mass[d], weight(z));
      });
      __syncthreads();
      // the largest digits first: two bins a thread
      const int bin = (1 << digits) - 1 - 2 * tid;
      unsigned long long v[2] = {0, 0};
      if (bin > 0) {
        v[0] = MASS ? s.mass[bin] : s.count[bin];
        v[1] = MASS ? s.mass[bin - 1] : s.count[bin - 1];
      }
      unsigned long long run = v[0] + v[1];
      for (int o = 1; o < 64; o *= 2) {
        const unsigned long long y = __shfl_up(run, o, 64);
        if (lane >= o) run += y;
      }
      if (lane == 63) s.sums[wave] = run;
      __syncthreads();
      unsigned long long all = 0, past = 0;
      for (int w = 0; w < WAVES; ++w) {
        past += w < wave ? s.sums[w] : 0;
        all += s.sums[w];
      }
      if (level == 0) target = target_of(all);
      past += run - v[0] - v[1];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (past < target && target <= past + v[i]) s.digit = bin - i, s.before = past;
        past += v[i];
      }
      __syncthreads();
      target -= s.before;
      prefix = prefix << digits | (unsigned)s.digit;
      const unsigned n = s.count[s.digit];
      const unsigned long long m = MASS ? s.mass[s.digit] : 0;
      __syncthreads();
      high = shift;
      if (high) continue;
      // n equal tokens: how many of them
      unsigned long long take = target;
      if (MASS) {
        const unsigned long long each = m / n;
        take = (target + each - 1) / each;
      }
      Cut cut{prefix, row.V};
      if (take < n)
        cut.index = first([&](int i, float z) -> unsigned long long { return key_of<T>(z) == prefix; },
                          [&](unsigned long long) { return take - 1; });
      cut.index = kept.key == prefix ? min(cut.index, kept.index) : cut.index;
      return cut;
    }
  }
};

template <typename T>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleArgs a) {
  __shared__ Lds s;
  const int64_t b = blockIdx.x;
  const pnfx_sampling& set = a.set;
  const double temperature = set.temperature_each ? (double)set.temperature_each[b] : set.temperature;
  const int64_t top_k = set.top_k_each ? (int64_t)set.top_k_each[b] : set.top_k;
  const double top_p = set.top_p_each ? (double)set.top_p_each[b] : set.top_p;
  const double min_p = set.min_p_each ? (double)set.min_p_each[b] : set.min_p;
  Sampler<T> me(static_cast<const T*>(a.z) + b * a.rs, a.V, s);
  if (me.tid < STEPS) s.table[me.tid] = exp2(me.tid * (1.0 / STEPS));
  float top = -__builtin_inff();
  bool nan = false;
  me.row.each(me.tid, me.row.chunks, THREADS, [&](int, float z) {
    top = fmaxf(top, z);
    nan |= z != z;
  });
  top = wave_max(top);
  nan = __any(nan);
  if (me.lane == 0) s.top[me.wave] = top, s.flag[me.wave] = nan;
  __syncthreads();
  for (int w = 0; w < WAVES; ++w) top = fmaxf(top, s.top[w]), nan |= s.flag[w] != 0;
  int token = -1;
  if (!nan && top > -__builtin_inff()) {
    if (!(temperature > 0) || top_k == 1) {
      token = me.first([&](int, float z) -> unsigned long long { return z == top; },
                       [](unsigned long long) { return 0ull; });
    } else {
      Weights w;
      w.table = s.table, w.zmax = top, w.S = a.S;
      w.c = fmin(STEPS * LOG2E / temperature, 1e300);
      w.low = min_p > 0 ? STEPS * log2(fmin(min_p, 1.0)) : -__builtin_inf();
      Cut cut{0, a.V};
      if (top_k > 0 && top_k < a.V)
        cut = me.template threshold<false>(cut, w, [&](unsigned long long) { return (unsigned long long)top_k; });
      if (top_p < 1)
        cut = me.template threshold<true>(cut, w, [&](unsigned long long all) {
          const double part = ceil(fmax(top_p, 0.0) * (double)all);
          return min(max((unsigned long long)part, 1ull), all);
        });
      const double u = fmin(fmax((double)a.u[b], 0.0), 1.0);
      token = me.first(
          [&](int i, float z) -> unsigned long long {
            if (!cut.keeps(key_of<T>(z), i)) return 0;
            const double y = w.steps(z);
            return y >= w.low ? w.of_steps(y) : 0;
          },
          [&](unsigned long long all) { return min((unsigned long long)(u * (double)all), all - 1); });
    }
  }
  if (me.tid == 0) a.tokens[b] = token;
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
  if (dtype == PNFX_F32) sample_kernel<float><<<dim3((unsigned)B), dim3(THREADS), 0, st>>>(a);
  else sample_kernel<bf16><<<dim3((unsigned)B), dim3(THREADS), 0, st>>>(a);
  return launch_status("sample");
}
