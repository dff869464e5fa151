// Softmax cross entropy of the logits z = x W^T (x [T, D], W [V, D]) against target tokens, without the logits:
//   lse_t = log sum_v exp z_tv,  loss_t = lse_t - z_t,target,  d_tv = (exp(z_tv - lse_t) - [v = target_t]) s_t,
//   dx = d W,  dW = d^T x,
// with s_t the loss's gradient of row t (1 / kept rows of it for a mean).
//
// Rows whose target is ignore_index are left out before anything else: xent_rows_kernel copies the others to
// the front of a buffer, so they cost no products, and what they hold, infinities included, reaches no sum.
//
// Forward: workgroups of one tile of rows each run over a range of the vocabulary and keep, in registers, the
// running maximum and the sum of exponentials of what each lane has seen; xent_loss_kernel joins them.  The
// target's logit is a dot product of its own.
//
// Backward: z is computed again for a piece of the vocabulary at a time (whose d, in the operands' type, is 256 MB
// or 2048 tokens' worth) and d is written in place of the logits; then dx += d W over the piece, in fp32, and
// the piece's rows of dW = d^T x.  bf16 operands: d is rounded to bf16 once, 2^-8 of each of its elements at
// most, as it is an operand of bf16 products.  It is rounded without s_t: the target's element, close to -1 for
// most rows, would otherwise be off by the same amount in each of them, and a frequent token's sum with it (0.4 % where
// 1 / rows rounds badly).  s_t enters the fp32 results where it is one value.  For a loss per row it enters dx's rows in
// fp32 and the x of dW = d^T (s x), which is rounded to bf16 with it, 2^-8 once more: the sum over rows leaves no
// place behind the product, and in d it would round the target's elements as above.  The target's own element is
// expm1(-loss_t), which keeps its digits where the softmax is close to one.
//
// Exponentials are taken in base 2, exp2(z L - m L) with L = log2 e as one fma per logit.  In the forward the rounding
// of m L is the same for a whole row and comes out again at its end, as the factor unround(m) = exp2(round(m L) - m L):
// without it logits around 5e4 would be 4e-3 off.  Beyond 2^24 logits are subtracted first.  In the backward m is the
// log-sum-exp, rounded to fp32, and the softmax is off by 2^-23 of it; rows for which that would show (kFarLse) are
// subtracted first, too, and what the rounding took from the log-sum-exp comes back from the loss: dot(x_t, W_target) +
// loss_t is the same number in two parts.  That leaves 2^-23 of the loss, or of the log-sum-exp where it is the smaller.
#include <algorithm>
#include <type_traits>

#include "product.h"

namespace pnfx {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float unround(float m) { return exp2_fast(-__builtin_fmaf(m, kLog2e, -(m * kLog2e))); }
// Beyond here the rounding of m L reaches whole units and, from about 2^30 on, more than an exponent holds: infinite or NaN
// sums for lanes whose logits so far are all the type's lowest value, say.  A workgroup that ends with such a maximum or sum
// goes through its tiles again and subtracts first.  (Tokens that are masked so cost that where they fill a lane's columns.)
constexpr float kFarTop = 16777216.f;
// The backward's |log-sum-exp| from which on a row is far: 2^-13 and 2^-18 of an element of the softmax.
template <typename T>
constexpr float kFarLse = sizeof(T) == 2 ? 1024.f : 32.f;
// Joins (top, sum) with (top2, sum2): maxima of logits and sums of exponentials beside them.  While nothing but
// -infinity was seen there is nothing to scale.
__device__ __forceinline__ void join(float& top, float& sum, float top2, float sum2) {
  const float next = fmaxf(top, top2), ref = next == -INFINITY ? 0.f : next;
  sum = sum * exp2_fast((top - ref) * kLog2e) + sum2 * exp2_fast((top2 - ref) * kLog2e);
  top = next;
}

// A lane's part of x . w; U loads on their way, the same bits for any U.
template <int U, typename T>
__device__ __forceinline__ float dot_part(const T* x, const T* w, int K, int lane) {
  float dot = 0.f;
#pragma unroll U
  for (int k = lane; k < K; k += 64) dot = __builtin_fmaf(to_f32(x[k]), to_f32(w[k]), dot);
  return dot;
}

// -------------------------------------------------------------------------- kept rows
constexpr int kRowsBlocks = 512;

struct RowsArgs {
  const void* x;
  const int64_t* target;
  void* xc;         // [T][Dp] kept rows, zero-padded
  int* pos;         // [T] place of a row among the kept ones, or -1
  int* tgt;         // [kept] target, or -1 where it is no token
  int* count;
  int64_t x_rs, ignore;
  int T, D, Dp, V, per;  // per: rows of a workgroup
  // backward only: row constants {lse, the rest of it times log2 e, expm1(-loss_t), target or -1}; s_t; it again where it is
  // one value; s_t x_t where not
  const void* w;
  int64_t ldw;
  const float* lse;
  const float* loss;
  const float* dloss;
  float4* rowc;
  float* s;
  int* far;  // of each workgroup: whether a row of its own is far
  float* alpha;
  void* xs;
  int reduction;
  bool vec;  // rows in whole, aligned 16-byte chunks
};

template <typename T>
__global__ __launch_bounds__(256) void xent_rows_kernel(RowsArgs a) {
  __shared__ int red[4];
  __shared__ int list[256];
  __shared__ float scale[256];
  __shared__ float2 stat[256];  // log-sum-exp, loss
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int r0 = blockIdx.x * a.per, r1 = min(r0 + a.per, a.T);
  // kept rows before this workgroup's, and (backward, for the mean) behind them
  int before = 0, total = 0;
  const int to = a.rowc ? a.T : r0;
  constexpr int U = 16;  // a thread's loads on their way (8 and single ones at the end: 15.3 against 14 us, T = 16384)
  for (int b = tid; b < to; b += 256 * U) {
    int64_t t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) t[u] = a.target[min(b + 256 * u, to - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = b + 256 * u, k = r < to && t[u] != a.ignore;
      total += k;
      before += r < r0 ? k : 0;
    }
  }
  const auto block_sum = [&](int v) {
    v = wave_sum_i(v);
    __syncthreads();
    if (lane == 0) red[wave] = v;
    __syncthreads();
    return red[0] + red[1] + red[2] + red[3];
  };
  before = block_sum(before);
  if (a.rowc) total = block_sum(total);
  float row_scale = 1.f;
  if (a.rowc && a.reduction != PNFX_REDUCE_NONE) {
    row_scale = a.reduction == PNFX_REDUCE_SUM ? a.dloss[0]
                : total ? a.dloss[0] / (float)total : 0.f;  // no rows: no gradients
    if (blockIdx.x == 0 && tid == 0) *a.alpha = row_scale;
  }
  bool far = false;
  for (int c0 = r0; c0 < r1; c0 += 256) {
    const int r = c0 + tid;
    const int64_t t = r < r1 ? a.target[r] : a.ignore;
    const bool keep = r < r1 && t != a.ignore;
    const uint64_t mask = __ballot(keep);
    __syncthreads();
    if (lane == 0) red[wave] = __popcll(mask);
    __syncthreads();
    int at = __popcll(mask & ((1ull << lane) - 1));
    for (int w = 0; w < wave; ++w) at += red[w];
    const int n = red[0] + red[1] + red[2] + red[3];
    if (keep) {
      const int i = before + at;
      const bool valid = t >= 0 && t < a.V;
      list[at] = r;
      a.tgt[i] = valid ? (int)t : -1;
      if (a.rowc) {
        const float s = a.reduction == PNFX_REDUCE_NONE ? a.dloss[r] : row_scale;
        // a target that is no token: its loss is NaN, and so are its gradients
        const float lse = valid ? a.lse[r] : __builtin_nanf(""), loss = a.loss[r];
        a.rowc[i] = float4{lse, 0.f, expm1f(-loss), __int_as_float(valid ? (int)t : -1)};
        a.s[i] = s;
        far |= fabsf(lse) > kFarLse<T>;
        scale[at] = s;
        stat[at] = float2{lse, loss};
      }
    }
    if (r < r1) a.pos[r] = keep ? before + at : -1;
    __syncthreads();
    for (int i = wave; i < n; i += 4) {
      const T* x = static_cast<const T*>(a.x) + (int64_t)list[i] * a.x_rs;
      T* y = static_cast<T*>(a.xc) + (int64_t)(before + i) * a.Dp;
      T* ys = a.xs ? static_cast<T*>(a.xs) + (int64_t)(before + i) * a.Dp : nullptr;
      const float s = scale[i];
      if (a.vec) {  // 16 bytes at a time
        typedef typename Elem<T>::Frag F;
#pragma unroll 4
        for (int c = lane * per16<T>; c < a.D; c += 64 * per16<T>) {
          F v = *reinterpret_cast<const F*>(x + c);
          *reinterpret_cast<F*>(y + c) = v;
          if (ys) {
#pragma unroll
            for (int e = 0; e < per16<T>; ++e) v[e] = from_f32<T>(to_f32(v[e]) * s);
            *reinterpret_cast<F*>(ys + c) = v;
          }
        }
      } else {
#pragma unroll 8
        for (int c = lane; c < a.Dp; c += 64) {
          const T v = c < a.D ? x[c] : (T)0.f;
          y[c] = v;
          if (ys) ys[c] = from_f32<T>(to_f32(v) * s);
        }
      }
    }
    if (a.rowc) {  // seldom: far rows (a target that is no token has a NaN here, and is not far)
      for (int i = wave; i < n; i += 4) {
        const float lse = stat[i].x, loss = stat[i].y;
        if (!(fabsf(lse) > kFarLse<T> && loss < 0.5f * fabsf(lse))) continue;
        const float dot = wave_sum(dot_part<1>(static_cast<const T*>(a.x) + (int64_t)list[i] * a.x_rs,
                                               static_cast<const T*>(a.w) + a.target[list[i]] * a.ldw, a.D, lane));
        if (lane == 0) a.rowc[before + i].y = ((dot - lse) + loss) * kLog2e;
      }
    }
    before += n;
  }
  if (a.rowc) {
    far = block_sum(far) != 0;
    if (tid == 0) a.far[blockIdx.x] = far;
  }
  if (r1 == a.T && tid == 0) *a.count = before;
}

// -------------------------------------------------------------------------- forward
struct FwdArgs {
  const void* xc;
  const void* w;
  float2* part;  // [T][splits * WN] running maximum and sum
  const int* count;
  int64_t ldx, ldw, K;
  int V, tn, splits, per;  // per: vocabulary tiles of a split
};

// The tiles' product: KS > 0: of that many steps of k at most, A's fragments in registers.
template <typename T, class C, int KS, int STORES>
struct Tiles : Thin<T, KS, C, STORES> {
  static constexpr int LDS = Thin<T, KS, C, STORES>::LDS;
  typedef Thin<T, KS, C, STORES> P;
  template <class Done>
  __device__ __forceinline__ static void go(typename P::StageA& sa, typename P::StageB& sb, int64_t, int tiles, T* sm,
                                            int wave, int lane, f32x4 (&acc)[P::MI][P::NJ], Done done) {
    P::run_tiles(sa, sb, tiles, sm, wave, lane, acc, done);
  }
};
template <typename T, class C, int STORES>
struct Tiles<T, C, 0, STORES> : Product<T, ROW, ROW, C> {
  static constexpr int LDS = lds_of<C>;
  typedef Product<T, ROW, ROW, C> P;
  template <class Done>
  __device__ __forceinline__ static void go(typename P::StageA& sa, typename P::StageB& sb, int64_t K, int tiles, T* sm,
                                            int wave, int lane, f32x4 (&acc)[P::MI][P::NJ], Done done) {
    P::run_tiles(sa, sb, (int)((K + k_step<T> - 1) / k_step<T>), tiles, sm, wave, lane, acc, done);
  }
};

template <typename T, class C, int KS>
__global__ __launch_bounds__(threads_of<C>, 2) void xent_fwd_kernel(FwdArgs a) {
  typedef Tiles<T, C, KS, 0> P;
  extern __shared__ __align__(16) char sm[];
  const int M = *a.count, tms = (M + C::TM - 1) / C::TM;
  if ((int)blockIdx.x >= tms * a.splits) return;
  int tm, split;
  tile_of(blockIdx.x, tms, a.splits, tm, split);
  const int m0 = tm * C::TM;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / C::WN * P::MI, wn = wave % C::WN * P::NJ;
  float top[P::MI], sum[P::MI];
  const int t0 = split * a.per, tiles = min(a.tn - t0, a.per);
  const auto pass = [&](auto far) {
    constexpr bool FAR = decltype(far)::value;
    // The second pass takes the loop over k (the same sums) and works its addresses out anew: with A's fragments in
    // registers, or its addresses kept over the first pass's loop, it spilled.
    typedef Tiles<T, C, FAR ? 0 : KS, 0> P;
    int tid = threadIdx.x;
    if (FAR) asm volatile("" : "+v"(tid));
    const int lane = tid & 63;
#pragma unroll
    for (int i = 0; i < P::MI; ++i) top[i] = -INFINITY, sum[i] = 0.f;
    typename P::StageA sa;
    typename P::StageB sb;
    sa.init(static_cast<const T*>(a.xc) + m0 * a.ldx, a.ldx, M - m0, a.K, tid);
    sb.init(static_cast<const T*>(a.w) + (int64_t)t0 * C::TN * a.ldw, a.ldw, a.V - t0 * C::TN, a.K, tid);
    f32x4 acc[P::MI][P::NJ] = {};
    P::go(sa, sb, a.K, tiles, reinterpret_cast<T*>(sm), wave, lane, acc, [&](int t) {
      const int n0 = (t0 + t) * C::TN;
      if (n0 + C::TN > a.V) {  // past the vocabulary
#pragma unroll
        for (int j = 0; j < P::NJ; ++j) {
          const int n = n0 + stage_row<ROW>(wn + j, 4 * (lane >> 4));
#pragma unroll
          for (int i = 0; i < P::MI; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (n + r >= a.V) acc[i][j][r] = -INFINITY;
        }
      }
#pragma unroll
      for (int i = 0; i < P::MI; ++i) {
        float m = acc[i][0][0];
#pragma unroll
        for (int j = 0; j < P::NJ; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) m = fmaxf(m, acc[i][j][r]);
        // While nothing but -infinity and NaN was seen there is nothing to scale; a sum that is NaN by then stays so.
        if constexpr (FAR) {
          const float next = fmaxf(top[i], m), ref = next == -INFINITY ? 0.f : next;
          float s = next == -INFINITY ? sum[i] : sum[i] * exp2_fast((top[i] - next) * kLog2e);
#pragma unroll
          for (int j = 0; j < P::NJ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) s += exp2_fast((acc[i][j][r] - ref) * kLog2e);
          top[i] = next;
          sum[i] = s;
          __builtin_amdgcn_sched_barrier(0);
          continue;
        }
        // The reference follows the maximum only once it is 8 behind (the exponentials stay below e^8), which after the
        // first tiles is hardly ever: 95 against 106 us at T = 16384, D = 64, V = 33278, 1.52 against 1.58 ms at T = 8192,
        // D = 4096, V = 32000.  With A's four steps in registers there is none left for the branch (16 spilled: 350
        // against 302 us at T = 16384, D = 256, V = 33278), and it follows at every tile.
        if (KS == 4 || __any(m > top[i] + 8.f)) {
#pragma clang fp contract(off)  // both products rounded as below, so that unround() of the last takes all of it out
          const float next = fmaxf(top[i], m);
          sum[i] = next == -INFINITY ? sum[i] : sum[i] * exp2_fast(top[i] * kLog2e - next * kLog2e);
          top[i] = next;
        }
        const float c = top[i] == -INFINITY ? 0.f : top[i] * kLog2e;
        float s = sum[i];
#pragma unroll
        for (int j = 0; j < P::NJ; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) s += exp2_fast(__builtin_fmaf(acc[i][j][r], kLog2e, -c));
        sum[i] = s;
        if (KS == 4) __builtin_amdgcn_sched_barrier(0);  // one row block at a time (285 against 277 us at the size above)
      }
    });
  };
  pass(std::false_type{});
  bool far = false;
#pragma unroll
  for (int i = 0; i < P::MI; ++i) far |= !(sum[i] < INFINITY) || (fabsf(top[i]) > kFarTop && top[i] != -INFINITY);
  // (the loop's last barrier has left the LDS free)
  int* const votes = reinterpret_cast<int*>(sm);
  far = __any(far);
  if (lane == 0) votes[wave] = far;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < C::WM * C::WN; ++v) far |= votes[v] != 0;
  if (far) {
    __syncthreads();
    pass(std::true_type{});
  } else {
#pragma unroll
    for (int i = 0; i < P::MI; ++i)
      if (top[i] != -INFINITY) sum[i] *= unround(top[i]);
  }
  // over the four lanes of a row
#pragma unroll
  for (int i = 0; i < P::MI; ++i) {
#pragma unroll
    for (int o = 16; o <= 32; o <<= 1)
      join(top[i], sum[i], __shfl_xor(top[i], o, 64), __shfl_xor(sum[i], o, 64));
    const int m = m0 + stage_row<ROW>(wm + i, lane & 15);
    if (lane < 16 && m < M) a.part[(int64_t)m * (a.splits * C::WN) + split * C::WN + wave % C::WN] = float2{top[i], sum[i]};
  }
}

struct LossArgs {
  const void* xc;
  const void* w;
  const float2* part;
  const int *pos, *tgt;
  float *rows, *lse;   // [T] loss and log-sum-exp of every row (ignored: 0)
  float* out;          // reduction none: [T]
  double* sums;        // per workgroup
  int64_t ldx, ldw;
  int T, K, parts, reduction, per;  // per: rows of a workgroup
};
// One wave per row: joins the row's partial statistics, forms the target's logit and the loss.
template <typename T>
__global__ __launch_bounds__(256) void xent_loss_kernel(LossArgs a) {
  __shared__ double red[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r0 = blockIdx.x * a.per, r1 = min(r0 + a.per, a.T);
  double total = 0;
  for (int r = r0 + wave; r < r1; r += 4) {
    const int i = a.pos[r];
    float loss = 0.f, lse = 0.f;
    if (i >= 0) {
      float top = -INFINITY, sum = 0.f;
      for (int p = lane; p < a.parts; p += 64) {
        const float2 v = a.part[(int64_t)i * a.parts + p];
        join(top, sum, v.x, v.y);
      }
      const int t = a.tgt[i];
      float dot = 0.f;
      if (t >= 0)
        dot = dot_part<8>(static_cast<const T*>(a.xc) + i * a.ldx, static_cast<const T*>(a.w) + t * a.ldw, a.K, lane);
      const float m = wave_max(top), ref = m == -INFINITY ? 0.f : m;
      sum = wave_sum(sum * exp2_fast((top - ref) * kLog2e));
      dot = wave_sum(dot);
      const float log_sum = __builtin_amdgcn_logf(sum) * kLn2;
      lse = m + log_sum;
      // of a softmax close to one the difference may round to below zero
      loss = t >= 0 ? (m - dot) + log_sum : __builtin_nanf("");
      loss = loss < 0.f ? 0.f : loss;
    }
    if (lane == 0) {
      a.rows[r] = loss;
      a.lse[r] = lse;
      if (a.reduction == PNFX_REDUCE_NONE) a.out[r] = loss;
    }
    total += loss;
  }
  if (a.reduction == PNFX_REDUCE_NONE) return;
  if (lane == 0) red[wave] = total;
  __syncthreads();
  if (threadIdx.x == 0) a.sums[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}
// The workgroups' sums in a fixed order.
__global__ __launch_bounds__(256) void xent_total_kernel(const double* sums, int n, const int* count, float* out,
                                                         int reduction) {
  __shared__ double red[4];
  double v = 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 256) v += sums[i];
  v = wave_sum_d(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0] + red[1] + red[2] + red[3];
  if (threadIdx.x == 0) *out = (float)(reduction == PNFX_REDUCE_MEAN ? v / *count : v);
}

// -------------------------------------------------------------------------- backward
struct GradArgs {
  const void* xc;
  const void* w;      // the piece's first row
  void* d;            // [T][ldd]
  const float4* rowc;
  const int *tgt, *count;
  int64_t ldx, ldw, K, ldd;
  int v0, P, tn, splits, per;  // the piece's first token, its tokens; column tiles of a workgroup
};

// Whether one of the wave's N rows from m0 on (of M) is far.
template <typename T, int N>
__device__ __forceinline__ bool any_far(const float4* rowc, int m0, int M, int lane) {
  bool far = false;
#pragma unroll
  for (int r = 0; r < N; r += 64) far |= fabsf(rowc[min(m0 + r + lane, M - 1)].x) > kFarLse<T>;
  return __any(far);
}

__device__ __forceinline__ void store16(__amdgpu_buffer_rsrc_t d, unsigned at, u32x4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(v, d, at, 0, 0);
}

template <typename T, class C, int KS>
__global__ __launch_bounds__(threads_of<C>, 2) void xent_grad_kernel(GradArgs a) {
  // 16-byte stores of a lane and tile
  constexpr int STORES = (C::TM / C::WM / 16) * (C::TN / C::WN / 16) * 4 / per16<T>;
  typedef Tiles<T, C, KS, STORES> P;
  extern __shared__ __align__(16) char sm[];
  const int M = *a.count, tms = (M + C::TM - 1) / C::TM;
  if ((int)blockIdx.x >= tms * a.splits) return;
  int tm, split;
  tile_of(blockIdx.x, tms, a.splits, tm, split);
  const int m0 = tm * C::TM;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave / C::WN * P::MI, wn = wave % C::WN * P::NJ;
  const int Pc = (a.P + 7) & ~7;  // columns past the piece, up to a whole chunk, are zero
  // of each row its log-sum-exp, its target's column in the piece, if it has one there, its target's element of d, and the
  // rest of the log-sum-exp (in LDS: there are no registers left for them beside A's fragments, and a read from global
  // memory waits for every load and store on its way); published by the loop's first barrier
  __shared__ float4 rows[C::TM];
  for (int r = threadIdx.x; r < C::TM; r += threads_of<C>) {
    const int m = min(m0 + r, M - 1);
    const float4 c = a.rowc[m];
    rows[r] = float4{c.x, __int_as_float(a.tgt[m] - a.v0), c.z, c.y};
  }
  const bool far = any_far<T, C::TM / C::WM>(a.rowc, m0 + 16 * wm, M, lane);
  const auto out = __builtin_amdgcn_make_buffer_rsrc(static_cast<T*>(a.d) + m0 * a.ldd, 0,
                                                     (int)(min(M - m0, C::TM) * a.ldd * sizeof(T)), 0x00027000);
  const unsigned ldb = (unsigned)(a.ldd * sizeof(T)), row = stage_row<ROW>(wm, lane & 15) * ldb;
  const int t0 = split * a.per, tiles = min(a.tn - t0, a.per);
  typename P::StageA sa;
  typename P::StageB sb;
  sa.init(static_cast<const T*>(a.xc) + m0 * a.ldx, a.ldx, M - m0, a.K, threadIdx.x);
  sb.init(static_cast<const T*>(a.w) + (int64_t)t0 * C::TN * a.ldw, a.ldw, a.P - t0 * C::TN, a.K, threadIdx.x);
  f32x4 acc[P::MI][P::NJ] = {};
  P::go(sa, sb, a.K, tiles, reinterpret_cast<T*>(sm), wave, lane, acc, [&](int t) {
    // the lane's first column; block j's are col(j) .. col(j) + 3 behind it
    const int n0 = (t0 + t) * C::TN, nl = n0 + 16 * wn + 8 * (lane >> 4);
    const auto col = [](int j) { return stage_row<ROW>(j, 0); };
    const bool edge = n0 + C::TN > a.P;
#pragma unroll
    for (int i = 0; i < P::MI; ++i) {
      const float4& row4 = rows[stage_row<ROW>(wm + i, lane & 15)];
      const float2 c{row4.x, row4.y};
      float l = c.x * kLog2e;
      if (far) {
#pragma unroll
        for (int j = 0; j < P::NJ; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] -= c.x;
        l = row4.w;
      }
#pragma unroll
      for (int j = 0; j < P::NJ; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[i][j][r] = exp2_fast(__builtin_fmaf(acc[i][j][r], kLog2e, -l));
      // 16 bytes at a time; the buffer's bounds drop the rows past M, a far offset the columns past the piece
      const unsigned at = row + stage_row<ROW>(i, 0) * ldb + nl * (unsigned)sizeof(T);
#pragma unroll
      for (int j = 0; j < P::NJ; j += 2) {
        float v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = acc[i][j + (r >> 2)][r & 3];
        unsigned o = at + col(j) * (unsigned)sizeof(T);
        if (edge) {
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (nl + col(j) + r >= a.P) v[r] = 0.f;
          if (nl + col(j) >= Pc) o = 0x80000000u;
        }
        if constexpr (sizeof(T) == 2) {
          store16(out, o, __builtin_bit_cast(u32x4, pack8(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7])));
        } else {
          store16(out, o, __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]}));
          store16(out, o + 16, __builtin_bit_cast(u32x4, f32x4{v[4], v[5], v[6], v[7]}));
        }
      }
      // seldom: the row's target is among the lane's columns; this store is the same thread's and comes later
      const int own = __float_as_int(c.y) - nl;
      if ((unsigned)own < 16u * P::NJ && (own & 24) == 0) {
        const T v = from_f32<T>(row4.z);
        if constexpr (sizeof(T) == 2)
          __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, v), out, at + own * 2, 0, 0);
        else
          __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), out, at + own * 4, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);  // one row block at a time: no registers for more
    }
  });
}

// Rows of at most 64 columns: the gradients without d in memory.  There the products are so short that writing d and
// reading it twice would be most of the time (xent_narrow, per 7936 tokens: 61 us for d, 105 for the two products).
// A workgroup keeps 128 rows of one operand, as fragments in registers, and goes through tiles of 128 rows
// of the other: the tile's logits, their exponentials, rounded to bf16 in the registers that are the next product's
// operand, and the product with the same tile, read transposed from where it lies in LDS.  For dx the rows kept are
// x's and the tiles W's; for dW the other way round, with the rows' log-sum-exps along the tile.
struct NarrowArgs {
  const void* a;    // rows kept, of lda
  const void* b;    // tiles, of ldb
  float* sums;      // [splits][M][N]: of a's rows
  const float4* rowc;
  const int *tgt, *count, *far;
  int64_t lda, ldb, K;
  int M, N, nb;     // rows of a and columns of the result (all of the array's); rows of b
  int V, splits, per;
  int blocks;       // of far
};
template <bool DW>
__global__ __launch_bounds__(256, 2) void xent_narrow_kernel(NarrowArgs a) {
  typedef Stage<bf16, ROW, 128, 256> St;
  constexpr int SB = 128 * 64, RING = 4;
  extern __shared__ __align__(16) char smem[];
  bf16* const sm = reinterpret_cast<bf16*>(smem);
  float4* const cols = reinterpret_cast<float4*>(smem + RING * SB * 2);  // DW: [RING][wave][64] of the tile's rows
  float4* const rowl = reinterpret_cast<float4*>(smem + RING * SB * 2);  // dx: [128] of the rows kept
  const int count = *a.count;
  const int rows = DW ? a.M : count, nb = DW ? count : a.nb;
  const int tms = (rows + 127) / 128;
  if ((int)blockIdx.x >= tms * a.splits) return;
  int tm, split;
  tile_of(blockIdx.x, tms, a.splits, tm, split);
  const int m0 = tm * 128, t0 = split * a.per, tiles = max(0, min((nb + 127) / 128 - t0, a.per));
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = wave >> 1, wn = wave & 1, r16 = lane & 15, g = lane >> 4;
  f32x4 out[4][4] = {};  // [row block][block of 16 columns of the result]
  const unsigned la = __builtin_amdgcn_readfirstlane(lds_addr(sm));
  if (tiles) {
    St sa, sb;
    sa.init(static_cast<const bf16*>(a.a) + m0 * a.lda, a.lda, rows - m0, a.K, threadIdx.x);
    sb.init(static_cast<const bf16*>(a.b) + (int64_t)t0 * 128 * a.ldb, a.ldb, nb - t0 * 128, a.K, threadIdx.x);
    const u32x4 dc = buffer_of(a.rowc, (unsigned)nb * 16u);
    const auto load = [&](int s) {
      sb.load(la + 2 * (s % RING) * SB, wave);
      sb.move(128, 1);
      if constexpr (DW)
        lds_dma16(dc, ((t0 + s) * 128 + 64 * wn + lane) * 16u, la + 2 * RING * SB + ((s % RING) * 4 + wave) * 1024);
    };
    constexpr int NI = St::NI + (DW ? 1 : 0);
    sa.load(la, wave);
    // whether any row is far, which takes another loop (a branch in the one for the others cost them up to 4 %)
    bool far = false;
    for (int b = threadIdx.x; b < a.blocks; b += 256) far |= a.far[b] != 0;
    int* const votes = reinterpret_cast<int*>(cols);
    far = __any(far);
    if (lane == 0) votes[wave] = far;
    wait_vm_lgkm<0>();
    __syncthreads();
#pragma unroll
    for (int v = 0; v < 4; ++v) far |= votes[v] != 0;
    bf16x8 fa[2][4];
    {
      const Frags<bf16, ROW> f(sm + wm * 64 * 64, lane);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int i = 0; i < 4; ++i) fa[hf][i] = f.get(i, hf, 0);
    }
    wait_vm_lgkm<0>();
    __syncthreads();
    // dx: each row's log-sum-exp, its target as a column of the first tile, the target's element, and the rest of the
    // log-sum-exp; published by the loop's first barrier
    if constexpr (!DW) {
      if (threadIdx.x < 128) {
        const int m = min(m0 + (int)threadIdx.x, rows - 1);
        const float4 c = a.rowc[m];
        rowl[threadIdx.x] = float4{c.x, __int_as_float(a.tgt[m] - t0 * 128), c.z, c.y};
      }
      wait_vm_lgkm<0>();
    }
    const Frags<bf16, ROW> fb(sm + wn * 64 * 64, lane);
    const Frags<bf16, COL> ft(sm + wn * 64 * 64, lane);
    load(0);
    if (tiles > 1) load(1);
    if (tiles > 2) load(2);
    const auto loop = [&](auto far) {
      constexpr bool FAR = decltype(far)::value;
      for (int t = 0; t < tiles; ++t) {
        const int buf = t % RING;
        if (t + 2 < tiles) wait_vm_lgkm<2 * NI>();
        else wait_vm_lgkm<0>();
        __builtin_amdgcn_s_barrier();
        if (t + 3 < tiles) load(t + 3);
        __builtin_amdgcn_sched_barrier(0);
        f32x4 z[4][4];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          bf16x8 b[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = fb.get(j, hf, buf * SB);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) z[i][j] = mma(b[j], fa[hf][i], hf ? z[i][j] : f32x4{});
        }
        const auto col = [](int j) { return stage_row<ROW>(j, 0); };  // block j's first column of the lane's
        const float4* const c = cols + (buf * 4 + wave) * 64;
        // Seldom a target's own element is among the wave's: which of its blocks have one.
        if constexpr (DW) {
          // (the log-sum-exps of the lane's 16 columns)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float4& c4 = c[8 * g + col(j) + r];
              const float lse = c4.x, l = FAR ? c4.y : lse * kLog2e;
#pragma unroll
              for (int i = 0; i < 4; ++i) z[i][j][r] = exp2_fast(__builtin_fmaf(FAR ? z[i][j][r] - lse : z[i][j][r], kLog2e, -l));
            }
          const uint64_t hits = __ballot((unsigned)(__float_as_int(c[lane].w) - m0 - 64 * wm) < 64u);
          if (hits) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (!(hits >> col(j) & 0x0f0f0f0fu)) continue;
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float4 e = c[8 * g + col(j) + r];
                const int own = __float_as_int(e.w) - m0 - 64 * wm;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (own == stage_row<ROW>(i, r16)) z[i][j][r] = e.z;
              }
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4& c = rowl[stage_row<ROW>(4 * wm + i, r16)];
            const float lse = c.x, l = FAR ? c.w : lse * kLog2e;
            const int at = __float_as_int(c.y) - 128 * t - 64 * wn - 8 * g;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                z[i][j][r] = exp2_fast(__builtin_fmaf(FAR ? z[i][j][r] - lse : z[i][j][r], kLog2e, -l));
            if (__any((unsigned)at < 40u)) {
              const float own = c.z;
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  if (at == col(j) + r) z[i][j][r] = own;
            }
          }
        }
        if (!DW && (t0 + t + 1) * 128 > a.V) {  // tokens past the vocabulary: of zero weights, but not finite perhaps
          const int n0 = (t0 + t) * 128 + 64 * wn + 8 * g;
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (n0 + col(j) + r >= a.V) {
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i][j][r] = 0.f;
              }
        }
        __builtin_amdgcn_sched_barrier(0);
        // two blocks: the lane's eight consecutive columns, a fragment of the next product
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          bf16x8 b[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = ft.get(j, h, buf * SB);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const f32x4 u = z[i][2 * h], v = z[i][2 * h + 1];
            const bf16x8 p = pack8(u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[i][j] = mma(b[j], p, out[i][j]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (far) loop(std::true_type{});
    else loop(std::false_type{});
    wait_vm_lgkm<0>();
  }
  // the two waves of a row share its columns of the tiles: their sums are added, half of them by each
  __syncthreads();
  f32x4* const other = reinterpret_cast<f32x4*>(smem) + wave * 512 + lane;
  const f32x4* const mine = reinterpret_cast<f32x4*>(smem) + (wave ^ 1) * 512 + lane;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) other[(4 * i + j) * 64] = wn ? out[i][j] : out[2 + i][j];
  __syncthreads();
  float* const sums = a.sums + (int64_t)split * a.M * a.N;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int m = m0 + stage_row<ROW>(4 * wm + 2 * wn + i, r16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4 v = (wn ? out[2 + i][j] : out[i][j]) + mine[(4 * i + j) * 64];
      const int n = 16 * j + 4 * g;
      if (m >= rows) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < a.N) sums[(int64_t)m * a.N + n + r] = v[r];
    }
  }
}
constexpr int kNarrowLds[2] = {4 * 128 * 128 + 128 * 16, 4 * 128 * 128 + 4 * 4 * 1024};  // dx, dW

struct DxArgs {
  const float* sums;  // [splits][T][D]
  const float* s;     // [kept]
  const int* pos;
  void* dx;           // [T][D]
  int64_t TD;
  int D, splits;
};
// dx in the operands' type: s_t times the splits' sums of a kept row, in split order, zeros for the others.
template <typename T>
__global__ __launch_bounds__(256) void xent_dx_kernel(DxArgs a) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = a.D % 4 == 0 ? 4 : 1;
  if (e * per >= a.TD) return;
  const int row = (int)(e * per / a.D), col = (int)(e * per % a.D), i = a.pos[row];
  T* dx = static_cast<T*>(a.dx) + e * per;
  const float* s = a.sums + (int64_t)i * a.D + col;
  if (per == 4) {
    f32x4 v = {};
    if (i >= 0)
      for (int p = 0; p < a.splits; ++p) v += *reinterpret_cast<const f32x4*>(s + p * a.TD);
    if (i >= 0) v *= a.s[i];
    if constexpr (sizeof(T) == 2) *reinterpret_cast<bf16x4*>(dx) = bf16x4{(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
    else *reinterpret_cast<f32x4*>(dx) = v;
  } else {
    float v = 0.f;
    if (i >= 0)
      for (int p = 0; p < a.splits; ++p) v += s[p * a.TD];
    if (i >= 0) v *= a.s[i];
    *dx = from_f32<T>(v);
  }
}

// -------------------------------------------------------------------------- host side
struct Sizes {
  int64_t T, D, V, Dp;
  int es, dtype;
};
Sizes sizes_of(int64_t T, int64_t D, int64_t V, int dtype) {
  return Sizes{T, D, V, round_up(D, 8), dtype == PNFX_F32 ? 4 : 2, dtype};
}
struct Arena {
  char* p;
  int64_t used;
  template <typename U>
  U* take(int64_t n) {
    char* r = p ? p + used : nullptr;
    used += round_up(n * (int64_t)sizeof(U), 256);
    return reinterpret_cast<U*>(r);
  }
};

// Whether logits are formed in tiles of 256.  The exponentials of such a tile are not hidden by a neighbour's products
// (128-tiles share a CU), so it pays where the products are long (us of the loss, tiles of 128 / 256, 8192 rows
// by 32768 tokens: D = 384 236 / 231, training 1063 / 1125; D = 512 294 / 273, 1116 / 1078; D = 1024 540 / 467, 2035 /
// 1866), there are tiles for every CU, and rounding the rows up to it costs little (333 rows by 50257 tokens, D = 1000:
// 70 / 75; 512 rows by 65536, D = 2048: 156 / 130).
bool big_tiles(const Sizes& z, int64_t tokens) {
  return z.dtype == PNFX_BF16 && z.D >= 512 && ceil_div(z.T, 256) * ceil_div(tokens, 256) >= 256 &&
         round_up(z.T, 256) * 4 <= round_up(z.T, 128) * 5;
}
// The forward's cut: tiles of rows by ranges of the vocabulary, two or more workgroups for each place on the chip.
struct FwdCut {
  bool big;
  int64_t tm, tn, splits, per;
};
// Vocabulary tiles that a workgroup goes through: 64 steps of k to pay for its start, less where that leaves
// fewer than four workgroups for each place on the chip.
int64_t tiles_per(const Sizes& z, int64_t tm, int64_t tn) {
  const int64_t steps = ceil_div(z.D * z.es, 128), most = std::max<int64_t>(1, tm * tn / 2048);
  return std::min(ceil_div(64, steps), most);
}
FwdCut fwd_cut(const Sizes& z) {
  FwdCut c;
  c.big = big_tiles(z, z.V);
  c.tm = ceil_div(z.T, c.big ? 256 : 128);
  c.tn = ceil_div(z.V, c.big ? 256 : 128);
  c.per = tiles_per(z, c.tm, c.tn);
  c.splits = ceil_div(c.tn, c.per);
  return c;
}
// Tokens of a piece: 256 MB of d.  Smaller pieces write and read dx's fp32 sums more often, larger ones take more memory;
// in between the time goes by how well the piece's two products divide, and not by its size.  Training calls, us, by the
// most that a piece may hold (MB): 16384 x 256 x 33278 128 1681, 160 1563, 192 1511, 224 1242, 256 1246, 320 1680, 384 1684,
// where 224 and 256 are the same five pieces and the only ones for which cut_group takes 256-tiles; 8192 x 2048 x 65536, with
// 256-tiles at each, 128 5825, 192 5993, 224 5855, 256 and 320, the same four pieces, 5706 and 5708, 384 5921.
int64_t piece_of(const Sizes& z) {
  const int64_t most = std::min(round_up(std::max<int64_t>((256ll << 20) / (z.T * z.es), 2048), 256), kMaxLd / 2);
  const int64_t n = ceil_div(z.V, most);
  return round_up(ceil_div(z.V, n), 256);
}

// Calls f(tile, steps) with the kernels' variant for this width: bf16 rows of up to 256 take Thin's.
template <typename T, class Fn>
int by_width(bool big, const Sizes& z, Fn f) {
  if constexpr (sizeof(T) == 2) {
    if (big) return f(Big{}, std::integral_constant<int, 0>{});
    if (z.Dp <= 64) return f(Mid{}, std::integral_constant<int, 1>{});
    if (z.Dp <= 128) return f(Mid{}, std::integral_constant<int, 2>{});
    if (z.Dp <= 192) return f(Mid{}, std::integral_constant<int, 3>{});
    if (z.Dp <= 256) return f(Mid{}, std::integral_constant<int, 4>{});
  }
  return f(Mid{}, std::integral_constant<int, 0>{});
}

struct Kept {
  void* xc;
  int *pos, *tgt, *count;
  void* w;  // padded copy, or null
};
Kept take_kept(Arena& ar, const Sizes& z, bool copy) {
  Kept k;
  k.xc = ar.take<char>(z.T * z.Dp * z.es);
  k.pos = ar.take<int>(z.T);
  k.tgt = ar.take<int>(z.T);
  k.count = ar.take<int>(1);
  k.w = copy ? ar.take<char>(z.V * z.Dp * z.es) : nullptr;
  return k;
}
int loss_rows_per(const Sizes& z) { return (int)std::max<int64_t>(4, ceil_div(z.T, 1024)); }
int64_t loss_blocks(const Sizes& z) { return ceil_div(z.T, loss_rows_per(z)); }

int64_t fwd_bytes(const Sizes& z, bool copy) {
  Arena ar{nullptr, 0};
  take_kept(ar, z, copy);
  const FwdCut c = fwd_cut(z);
  ar.take<float2>(c.splits * 4 * z.T);
  ar.take<double>(loss_blocks(z));
  return ar.used;
}
struct BwdCut {
  int64_t P;
  Cut dx, dw;
};
BwdCut bwd_cut(const Sizes& z) {
  BwdCut c;
  c.P = std::min(piece_of(z), round_up(z.V, 8));
  const Shape s[2] = {{z.T, z.D, c.P, true}, {c.P, z.D, z.T, false}};
  Cut cuts[2];
  cut_group(s, 2, z.dtype, true, cuts);
  c.dx = cuts[0], c.dw = cuts[1];
  return c;
}
// The narrow kernels' cut: parts of the tiles for each 128 rows kept, so that the last round of workgroups, two on a
// CU, is nearly full, against the fp32 sums that each part writes and another kernel reads.
struct NarrowCut {
  int64_t splits, per;
};
NarrowCut narrow_cut(int64_t rows, int64_t tiles, int64_t D) {
  const int64_t tm = ceil_div(rows, 128);
  NarrowCut best{1, tiles};
  double best_us = 1e30;
  for (int64_t s = 1; s <= std::min<int64_t>(32, tiles); ++s) {
    const int64_t per = ceil_div(tiles, s);
    const double us = ceil_div(tm * ceil_div(tiles, per), 512) * (per * 2.5 + 6.0) + ceil_div(tiles, per) * rows * D * 8 / 4e6;
    if (us < best_us) best_us = us, best = NarrowCut{ceil_div(tiles, per), per};
  }
  return best;
}
bool narrow(const Sizes& z, int reduction) {
  return z.dtype == PNFX_BF16 && z.Dp <= 64 && reduction != PNFX_REDUCE_NONE;
}
int64_t bwd_bytes(const Sizes& z, int reduction, bool copy) {
  Arena ar{nullptr, 0};
  take_kept(ar, z, copy);
  if (narrow(z, reduction)) {
    ar.take<float>(1);
    ar.take<float>(z.T);
    ar.take<int>(kRowsBlocks);
    ar.take<float4>(z.T);
    ar.take<float>(narrow_cut(z.T, ceil_div(z.V, 128), z.D).splits * z.T * z.D);
    ar.take<float>(narrow_cut(z.V, ceil_div(z.T, 128), z.D).splits * z.V * z.D);
    return ar.used;
  }
  ar.take<float>(1);
  ar.take<float>(z.T);
  ar.take<int>(kRowsBlocks);
  if (reduction == PNFX_REDUCE_NONE) ar.take<char>(z.T * z.Dp * z.es);  // s x
  const BwdCut c = bwd_cut(z);
  ar.take<float4>(z.T);
  ar.take<char>(z.T * c.P * z.es);
  ar.take<float>(c.dx.splits * z.T * z.D);
  ar.take<char>(product_workspace(c.dw, c.P, z.D));
  return ar.used;
}

// Workgroups of xent_rows_kernel and their rows.
int64_t rows_per(const Sizes& z) { return std::max<int64_t>(4, ceil_div(z.T, kRowsBlocks)); }
int64_t rows_blocks(const Sizes& z) { return ceil_div(z.T, rows_per(z)); }

template <typename T>
int keep_rows(const Kept& k, const void* x, int64_t x_rs, const int64_t* target, int64_t ignore, const Sizes& z,
              RowsArgs a, hipStream_t st) {
  a.x = x, a.target = target, a.xc = k.xc, a.pos = k.pos, a.tgt = k.tgt, a.count = k.count;
  a.x_rs = x_rs, a.ignore = ignore;
  a.T = (int)z.T, a.D = (int)z.D, a.Dp = (int)z.Dp, a.V = (int)z.V;
  a.per = (int)rows_per(z);
  a.vec = z.D == z.Dp && operand_ok(x, x_rs, z.es);
  return launch<xent_rows_kernel<T>>(rows_blocks(z), 256, 0, a, st, "xent rows");
}
// W in place, or its padded copy.
int take_w(const Kept& k, const void*& w, int64_t& w_rs, const Sizes& z, hipStream_t st) {
  if (!k.w) return PNFX_OK;
  const PadItem p{w, k.w, w_rs, z.V, z.D, z.V, z.Dp, 1};
  PNFX_TRY(pad(&p, 1, z.dtype, st));
  w = k.w, w_rs = z.Dp;
  return PNFX_OK;
}

template <typename T>
int xent_fwd(const void* x, int64_t x_rs, const void* w, int64_t w_rs, const int64_t* target, int64_t ignore,
             float* out, float* rows, float* lse, int reduction, const Sizes& z, bool copy, void* ws, hipStream_t st) {
  Arena ar{static_cast<char*>(ws), 0};
  const Kept k = take_kept(ar, z, copy);
  const FwdCut c = fwd_cut(z);
  float2* part = ar.take<float2>(c.splits * 4 * z.T);
  double* sums = ar.take<double>(loss_blocks(z));
  PNFX_TRY(take_w(k, w, w_rs, z, st));
  PNFX_TRY(keep_rows<T>(k, x, x_rs, target, ignore, z, RowsArgs{}, st));
  FwdArgs f{k.xc, w, part, k.count, z.Dp, w_rs, z.Dp, (int)z.V, (int)c.tn, (int)c.splits, (int)c.per};
  const int wn = c.big ? Big::WN : Mid::WN;
  PNFX_TRY((by_width<T>(c.big, z, [&](auto cfg, auto ks) {
    typedef decltype(cfg) C;
    constexpr int KS = decltype(ks)::value;
    return launch<xent_fwd_kernel<T, C, KS>>(c.tm * c.splits, threads_of<C>, Tiles<T, C, KS, 0>::LDS, f, st, "xent_fwd");
  })));
  LossArgs l{k.xc, w, part, k.pos, k.tgt, rows, lse, out, sums, z.Dp, w_rs,
             (int)z.T, (int)z.D, (int)c.splits * wn, reduction, loss_rows_per(z)};
  PNFX_TRY((launch<xent_loss_kernel<T>>(loss_blocks(z), 256, 0, l, st, "xent_loss")));
  if (reduction == PNFX_REDUCE_NONE) return PNFX_OK;
  hipLaunchKernelGGL(xent_total_kernel, dim3(1), dim3(256), 0, st, sums, (int)loss_blocks(z), k.count, out, reduction);
  return launch_status("xent_total");
}

template <typename T>
int xent_bwd(const float* dloss, const void* x, int64_t x_rs, const void* w, int64_t w_rs, const int64_t* target,
             int64_t ignore, const float* rows, const float* lse, void* dx, void* dw, int reduction, const Sizes& z,
             bool copy, void* ws, hipStream_t st) {
  Arena ar{static_cast<char*>(ws), 0};
  const Kept k = take_kept(ar, z, copy);
  RowsArgs r = {};
  r.lse = lse, r.loss = rows, r.dloss = dloss, r.reduction = reduction;
  r.alpha = ar.take<float>(1);
  r.s = ar.take<float>(z.T);
  r.far = ar.take<int>(kRowsBlocks);
  if constexpr (sizeof(T) == 2) {
    if (narrow(z, reduction)) {
      r.rowc = ar.take<float4>(z.T);
      const NarrowCut cx = narrow_cut(z.T, ceil_div(z.V, 128), z.D), cw = narrow_cut(z.V, ceil_div(z.T, 128), z.D);
      float* sx = ar.take<float>(cx.splits * z.T * z.D);
      float* sw = ar.take<float>(cw.splits * z.V * z.D);
      PNFX_TRY(take_w(k, w, w_rs, z, st));
      r.w = w, r.ldw = w_rs;
      PNFX_TRY(keep_rows<T>(k, x, x_rs, target, ignore, z, r, st));
      if (dx) {
        const NarrowArgs n{k.xc, w, sx, r.rowc, k.tgt, k.count, r.far, z.Dp, w_rs, z.Dp, (int)z.T, (int)z.D, (int)z.V,
                           (int)z.V, (int)cx.splits, (int)cx.per, (int)rows_blocks(z)};
        PNFX_TRY((launch<xent_narrow_kernel<false>>(ceil_div(z.T, 128) * cx.splits, 256, kNarrowLds[0], n, st, "xent_dx")));
        const DxArgs x1{sx, r.s, k.pos, dx, z.T * z.D, (int)z.D, (int)cx.splits};
        PNFX_TRY((launch<xent_dx_kernel<T>>(ceil_div(x1.TD, z.D % 4 == 0 ? 1024 : 256), 256, 0, x1, st, "xent_dx")));
      }
      if (dw) {
        const NarrowArgs n{w, k.xc, sw, r.rowc, k.tgt, k.count, r.far, w_rs, z.Dp, z.Dp, (int)z.V, (int)z.D, (int)z.T,
                           (int)z.V, (int)cw.splits, (int)cw.per, (int)rows_blocks(z)};
        PNFX_TRY((launch<xent_narrow_kernel<true>>(ceil_div(z.V, 128) * cw.splits, 256, kNarrowLds[1], n, st, "xent_dw")));
        PNFX_TRY(sum_splits(sw, (int)cw.splits, z.V, z.D, dw, r.alpha, z.dtype, st));
      }
      return PNFX_OK;
    }
  }
  const BwdCut c = bwd_cut(z);
  if (reduction == PNFX_REDUCE_NONE) r.xs = ar.take<char>(z.T * z.Dp * z.es);
  r.rowc = ar.take<float4>(z.T);
  T* d = reinterpret_cast<T*>(ar.take<char>(z.T * c.P * z.es));
  float* sums = ar.take<float>(c.dx.splits * z.T * z.D);
  void* dw_ws = ar.take<char>(product_workspace(c.dw, c.P, z.D));
  PNFX_TRY(take_w(k, w, w_rs, z, st));
  r.w = w, r.ldw = w_rs;
  PNFX_TRY(keep_rows<T>(k, x, x_rs, target, ignore, z, r, st));
  for (int64_t v0 = 0; v0 < z.V; v0 += c.P) {
    const int64_t n = std::min(c.P, z.V - v0);
    const T* wp = static_cast<const T*>(w) + v0 * w_rs;
    GradArgs g{k.xc, wp, d, r.rowc, k.tgt, k.count, z.Dp, w_rs, z.Dp, c.P, (int)v0, (int)n, 0, 0, 0};
    const bool big = big_tiles(z, n);
    const int64_t tm = ceil_div(z.T, big ? 256 : 128);
    g.tn = (int)ceil_div(round_up(n, 8), big ? 256 : 128);
    g.per = (int)tiles_per(z, tm, g.tn);
    g.splits = (int)ceil_div(g.tn, g.per);
    PNFX_TRY((by_width<T>(big, z, [&](auto cfg, auto ks) {
      typedef decltype(cfg) C;
      constexpr int KS = decltype(ks)::value;
      return launch<xent_grad_kernel<T, C, KS>>(tm * g.splits, threads_of<C>, Tiles<T, C, KS, 0>::LDS, g, st,
                                                "xent_grad");
    })));
    Job jobs[2];
    int nj = 0;
    if (dx) {
      ProductArgs p = {};
      p.a = d, p.b = wp, p.lda = c.P, p.ldb = w_rs, p.M = z.T, p.N = z.D, p.K = n;
      p.m_count = k.count, p.sums = sums, p.add = v0 > 0;
      jobs[nj++] = Job{ROW, COL, p, c.dx, nullptr};
    }
    if (dw) {
      ProductArgs p = {};
      p.a = d, p.b = r.xs ? r.xs : k.xc, p.c = static_cast<T*>(dw) + v0 * z.D, p.lda = c.P, p.ldb = z.Dp, p.ldc = z.D;
      p.M = n, p.N = z.D, p.K = z.T, p.k_count = k.count;
      p.alpha = r.xs ? nullptr : r.alpha;
      jobs[nj++] = Job{COL, COL, p, c.dw, dw_ws};
    }
    if (nj) PNFX_TRY(products(jobs, nj, z.dtype, st));
  }
  if (!dx) return PNFX_OK;
  const DxArgs x1{sums, r.s, k.pos, dx, z.T * z.D, (int)z.D, c.dx.splits};
  return launch<xent_dx_kernel<T>>(ceil_div(x1.TD, z.D % 4 == 0 ? 1024 : 256), 256, 0, x1, st, "xent_dx");
}

int check_sizes(const char* what, int64_t T, int64_t D, int64_t V, int reduction, int dtype) {
  PNFX_REQUIRE(dtype == PNFX_F32 || dtype == PNFX_BF16, "%s: unsupported dtype %d", what, dtype);
  PNFX_REQUIRE(reduction == PNFX_REDUCE_NONE || reduction == PNFX_REDUCE_SUM || reduction == PNFX_REDUCE_MEAN,
               "%s: unknown reduction %d", what, reduction);
  PNFX_REQUIRE(T >= 1 && D >= 1 && V >= 1 && T <= (1 << 24) && D <= (1 << 18) && V <= (1 << 24),
               "%s: bad shape T=%lld D=%lld V=%lld", what, (long long)T, (long long)D, (long long)V);
  return PNFX_OK;
}
bool copies_w(const void* w, int64_t w_rs, const Sizes& z) { return !(z.D == z.Dp && operand_ok(w, w_rs, z.es)); }

}  // namespace
}  // namespace pnfx

extern "C" int64_t pnfx_xent_fwd_workspace_size(int64_t T, int64_t D, int64_t V, int copies, int dtype) {
  using namespace pnfx;
  if (check_sizes("xent", T, D, V, PNFX_REDUCE_NONE, dtype) != PNFX_OK) return 0;
  return fwd_bytes(sizes_of(T, D, V, dtype), copies);
}
extern "C" int64_t pnfx_xent_bwd_workspace_size(int64_t T, int64_t D, int64_t V, int reduction, int copies, int dtype) {
  using namespace pnfx;
  if (check_sizes("xent", T, D, V, reduction, dtype) != PNFX_OK) return 0;
  return bwd_bytes(sizes_of(T, D, V, dtype), reduction, copies);
}

extern "C" int pnfx_xent_fwd(const void* x, int64_t x_rs, const void* w, int64_t w_rs, const int64_t* target,
                             int64_t ignore_index, float* loss, float* loss_rows, float* lse, int64_t T, int64_t D,
                             int64_t V, int reduction, int dtype, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  using namespace pnfx;
  PNFX_REQUIRE(x && w && target && loss && loss_rows && lse, "xent_fwd: null pointer");
  PNFX_TRY(check_sizes("xent_fwd", T, D, V, reduction, dtype));
  PNFX_REQUIRE(x_rs >= D && w_rs >= D, "xent_fwd: row strides %lld, %lld", (long long)x_rs, (long long)w_rs);
  const Sizes z = sizes_of(T, D, V, dtype);
  const bool copy = copies_w(w, w_rs, z);
  const int64_t need = fwd_bytes(z, copy);
  PNFX_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= need,
               "xent_fwd: workspace needs %lld bytes", (long long)need);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return dtype == PNFX_F32 ? xent_fwd<float>(x, x_rs, w, w_rs, target, ignore_index, loss, loss_rows, lse, reduction, z,
                                             copy, workspace, st)
                           : xent_fwd<bf16>(x, x_rs, w, w_rs, target, ignore_index, loss, loss_rows, lse, reduction, z,
                                            copy, workspace, st);
}

extern "C" int pnfx_xent_bwd(const float* dloss, const void* x, int64_t x_rs, const void* w, int64_t w_rs,
                             const int64_t* target, int64_t ignore_index, const float* loss_rows, const float* lse,
                             void* dx, void* dw, int64_t T, int64_t D, int64_t V, int reduction, int dtype,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace pnfx;
  PNFX_REQUIRE(dloss && x && w && target && loss_rows && lse, "xent_bwd: null pointer");
  PNFX_TRY(check_sizes("xent_bwd", T, D, V, reduction, dtype));
  PNFX_REQUIRE(x_rs >= D && w_rs >= D, "xent_bwd: row strides %lld, %lld", (long long)x_rs, (long long)w_rs);
  PNFX_REQUIRE(((reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(dw)) & 15) == 0,
               "xent_bwd: gradients must be 16-byte aligned");
  const Sizes z = sizes_of(T, D, V, dtype);
  const bool copy = copies_w(w, w_rs, z);
  const int64_t need = bwd_bytes(z, reduction, copy);
  PNFX_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= need,
               "xent_bwd: workspace needs %lld bytes", (long long)need);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return dtype == PNFX_F32 ? xent_bwd<float>(dloss, x, x_rs, w, w_rs, target, ignore_index, loss_rows, lse, dx, dw,
                                             reduction, z, copy, workspace, st)
                           : xent_bwd<bf16>(dloss, x, x_rs, w, w_rs, target, ignore_index, loss_rows, lse, dx, dw,
                                            reduction, z, copy, workspace, st);
}
