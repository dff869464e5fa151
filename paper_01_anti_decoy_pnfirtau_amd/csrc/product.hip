// Plain matrix products, the sum of their splits, and zero-padded copies.  What bounds the products and how they
// are staged: gemm.h.
#include "product.h"

namespace pnfx {
namespace {

struct MmArgs {
  const void *a, *b;
  void* c;
  float* sums;
  int64_t lda, ldb, ldc, K, steps;
  int M, N, tm, tn, splits;
  int gap_at, gap;
  const int *m_count, *k_count;
  const float* alpha;
  bool add;
};

// Row of C of product row m, or -1.
__device__ __forceinline__ int out_row(int m, int gap_at, int gap) {
  if (m < gap_at) return m;
  return m < gap_at + gap ? -1 : m - gap;
}

// Four columns from n on of a row of `N`, vectors where the row allows them.
template <typename T>
__device__ __forceinline__ void store4(T* row, int n, int N, bool aligned, f32x4 v) {
  if (aligned && n + 4 <= N) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4*>(row + n) = v;
    } else {
      *reinterpret_cast<bf16x4*>(row + n) = bf16x4{(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
    }
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < N) row[n + r] = from_f32<T>(v[r]);
  }
}

template <typename T, Kind KA, Kind KB, class C>
__global__ __launch_bounds__(threads_of<C>, 2) void mm_kernel(MmArgs g) {
  typedef Product<T, KA, KB, C> P;
  extern __shared__ __align__(16) char sm[];
  const int split = blockIdx.x / (g.tm * g.tn);
  int tm, tn;
  tile_of(blockIdx.x - split * g.tm * g.tn, g.tm, g.tn, tm, tn);
  const int m0 = tm * C::TM, n0 = tn * C::TN;
  const int M = g.m_count ? min(g.M, *g.m_count) : g.M;
  if (m0 >= M) return;
  const int64_t K = g.k_count ? min<int64_t>(g.K, *g.k_count) : g.K;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t k0 = split * g.steps * k_step<T>;
  const int64_t ks = min<int64_t>(K - k0, g.steps * k_step<T>);
  typename P::StageA sa;
  typename P::StageB sb;
  const T* a = static_cast<const T*>(g.a) + (KA == COL ? k0 * g.lda + m0 : m0 * g.lda + k0);
  const T* b = static_cast<const T*>(g.b) + (KB == COL ? k0 * g.ldb + n0 : n0 * g.ldb + k0);
  sa.init(a, g.lda, M - m0, ks, threadIdx.x);
  sb.init(b, g.ldb, g.N - n0, ks, threadIdx.x);
  f32x4 acc[P::MI][P::NJ] = {};
  P::run(sa, sb, (int)((ks + k_step<T> - 1) / k_step<T>), reinterpret_cast<T*>(sm), wave, lane, acc);
  const int wm = wave / C::WN * P::MI, wn = wave % C::WN * P::NJ;
  float* sums = g.sums ? g.sums + (int64_t)split * g.M * g.N : nullptr;
  const bool aligned = g.ldc % 4 == 0;
  const float alpha = g.alpha ? *g.alpha : 1.f;
#pragma unroll
  for (int i = 0; i < P::MI; ++i) {
    const int m = m0 + stage_row<KA>(wm + i, lane & 15);
    if (m >= M) continue;
    const int row = out_row(m, g.gap_at, g.gap);
#pragma unroll
    for (int j = 0; j < P::NJ; ++j) {
      const int n = n0 + stage_row<KB>(wn + j, 4 * (lane >> 4));
      if (n >= g.N) continue;
      if (sums) {
        float* s = sums + (int64_t)m * g.N + n;
        if (g.N % 4 == 0) {
          f32x4* s4 = reinterpret_cast<f32x4*>(s);
          *s4 = g.add ? *s4 + acc[i][j] : acc[i][j];
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n + r < g.N) s[r] = g.add ? s[r] + acc[i][j][r] : acc[i][j][r];
        }
      } else if (row >= 0) {
        store4<T>(static_cast<T*>(g.c) + row * g.ldc, n, g.N, aligned, acc[i][j] * alpha);
      }
    }
  }
}

struct SumArgs {
  const float* sums;
  void* c;
  const float* alpha;
  int64_t MN, ldc;
  int N, splits, gap_at, gap;
};
// C from the splits' sums, added in split order: four elements per thread.
template <typename T>
__global__ __launch_bounds__(256) void mm_sum_kernel(SumArgs g) {
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (e >= g.MN) return;
  const float alpha = g.alpha ? *g.alpha : 1.f;
  if (g.N % 4 == 0) {
    f32x4 acc = *reinterpret_cast<const f32x4*>(g.sums + e);
#pragma unroll 4
    for (int s = 1; s < g.splits; ++s) acc += *reinterpret_cast<const f32x4*>(g.sums + s * g.MN + e);
    const int row = out_row((int)(e / g.N), g.gap_at, g.gap);
    if (row >= 0)
      store4<T>(static_cast<T*>(g.c) + row * g.ldc, (int)(e % g.N), g.N, g.ldc % 4 == 0, acc * alpha);
    return;
  }
  for (int64_t i = e; i < min<int64_t>(e + 4, g.MN); ++i) {
    float acc = g.sums[i];
    for (int s = 1; s < g.splits; ++s) acc += g.sums[s * g.MN + i];
    const int row = out_row((int)(i / g.N), g.gap_at, g.gap);
    if (row >= 0) static_cast<T*>(g.c)[row * g.ldc + i % g.N] = from_f32<T>(acc * alpha);
  }
}

constexpr int kMaxPads = 4;
struct PadArgs {
  PadItem item[kMaxPads];
  int64_t first[kMaxPads + 1];  // workgroups of 4 rows each
  int n;
};
// One wave per row.
template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(PadArgs g) {
  int i = 0;
  while (i + 1 < g.n && (int64_t)blockIdx.x >= g.first[i + 1]) ++i;
  const PadItem& p = g.item[i];
  const int64_t r = (blockIdx.x - g.first[i]) * 4 + (threadIdx.x >> 6);
  if (r >= p.rows_out * p.halves) return;
  const int64_t half = r / p.rows_out, in = r % p.rows_out;
  const T* src = static_cast<const T*>(p.src) + (half * p.rows + in) * p.ld;
  T* dst = static_cast<T*>(p.dst) + r * p.cols_out;
  for (int64_t c = threadIdx.x & 63; c < p.cols_out; c += 64)
    dst[c] = in < p.rows && c < p.cols ? src[c] : (T)0.f;
}

template <typename T, Kind KA, Kind KB, class C>
int mm_launch(const MmArgs& g, hipStream_t st) {
  return launch<mm_kernel<T, KA, KB, C>>((int64_t)g.tm * g.tn * g.splits, threads_of<C>, lds_of<C>, g, st, "product");
}
template <typename T, class C>
int mm_kinds(int ka, int kb, const MmArgs& g, hipStream_t st) {
  if (ka == ROW && kb == ROW) return mm_launch<T, ROW, ROW, C>(g, st);
  if (ka == ROW && kb == COL) return mm_launch<T, ROW, COL, C>(g, st);
  PNFX_REQUIRE(ka == COL && kb == COL, "product: operands %d, %d", ka, kb);
  return mm_launch<T, COL, COL, C>(g, st);
}

}  // namespace

// The cut that is expected to be done first.  A tile's step takes, with one of its kind on every CU, the time of
// its products at the rate that gemm.h's figures give; a split adds its fp32 sums' way to memory and back.
Cut cut_of(int64_t M, int64_t N, int64_t K, int dtype, bool can_split) {
  const int es = dtype == PNFX_F32 ? 4 : 2;
  const int64_t steps = ceil_div(K, 128 / es);
  Cut best{false, 1, steps};
  double best_us = 1e30;
  for (int big = 0; big < (dtype == PNFX_BF16 ? 2 : 1); ++big) {
    const int64_t T = big ? 256 : 128, tiles = ceil_div(M, T) * ceil_div(N, T);
    // us of one step of a tile alone on its CU, and of the CU's tiles together
    const double rate = dtype == PNFX_F32 ? 110e6 : big ? 1300e6 : 1050e6;  // operations per us on 256 CUs
    const int per_cu = big ? 1 : 2;
    const double step_us = 2.0 * T * T * (128 / es) / (rate / 256) * per_cu;
    for (int64_t s = 1; s <= 64; s *= 2) {
      if (s > 1 && (!can_split || steps / s < 4)) break;
      const int64_t per = ceil_div(steps, s), slots = 256 * per_cu;
      const int64_t full = tiles * s / slots, rest = tiles * s % slots;
      // a last round that leaves CUs with one tile of two runs it faster
      const double last = !rest ? 0 : per_cu == 2 && rest <= 256 ? 0.9 : 1;
      double us = (full + last) * (per * step_us + 2.0);
      if (s > 1) us += 4.0 + s * M * N * 8 / 4e6;
      if (us < best_us) {
        best_us = us;
        best = Cut{big != 0, (int)ceil_div(steps, per), per};
      }
    }
  }
  return best;
}

int64_t product_workspace(const Cut& cut, int64_t M, int64_t N) {
  return cut.splits > 1 ? cut.splits * M * N * 4 : 0;
}

int product(int ka, int kb, const ProductArgs& p, const Cut& cut, int dtype, void* workspace, hipStream_t st) {
  if (p.M < 1 || p.N < 1) return PNFX_OK;
  const int es = dtype == PNFX_F32 ? 4 : 2;
  PNFX_REQUIRE(operand_ok(p.a, p.lda, es) && operand_ok(p.b, p.ldb, es), "product: operand alignment");
  PNFX_REQUIRE(p.M < (1 << 30) && p.N < (1 << 30) && p.K < (1ll << 31), "product: %lld x %lld over %lld",
               (long long)p.M, (long long)p.N, (long long)p.K);
  const bool summed = !p.sums && cut.splits > 1;
  PNFX_REQUIRE(!summed || workspace, "product: no workspace");
  const int64_t T = cut.big ? 256 : 128;
  MmArgs g;
  g.a = p.a;
  g.b = p.b;
  g.c = p.c;
  g.sums = summed ? static_cast<float*>(workspace) : p.sums;
  g.lda = p.lda;
  g.ldb = p.ldb;
  g.ldc = p.ldc;
  g.K = p.K;
  g.steps = cut.steps;
  g.M = (int)p.M;
  g.N = (int)p.N;
  g.tm = (int)ceil_div(p.M, T);
  g.tn = (int)ceil_div(p.N, T);
  g.splits = cut.splits;
  g.gap_at = p.gap ? (int)p.gap_at : (int)p.M;
  g.gap = (int)p.gap;
  g.m_count = p.m_count;
  g.k_count = p.k_count;
  g.add = p.add;
  g.alpha = summed ? nullptr : p.alpha;
  if (dtype == PNFX_F32)
    PNFX_TRY((mm_kinds<float, Mid>(ka, kb, g, st)));
  else if (cut.big)
    PNFX_TRY((mm_kinds<bf16, Big>(ka, kb, g, st)));
  else
    PNFX_TRY((mm_kinds<bf16, Mid>(ka, kb, g, st)));
  if (!summed) return PNFX_OK;
  SumArgs s{g.sums, p.c, p.alpha, p.M * p.N, p.ldc, g.N, cut.splits, g.gap_at, g.gap};
  const int64_t grid = ceil_div(s.MN, 1024);
  return dtype == PNFX_F32 ? launch<mm_sum_kernel<float>>(grid, 256, 0, s, st, "product sums")
                           : launch<mm_sum_kernel<bf16>>(grid, 256, 0, s, st, "product sums");
}

int pad(const PadItem* items, int n, int dtype, hipStream_t st) {
  if (!n) return PNFX_OK;
  PadArgs g;
  g.n = n;
  g.first[0] = 0;
  for (int i = 0; i < n; ++i) {
    g.item[i] = items[i];
    g.first[i + 1] = g.first[i] + ceil_div(items[i].rows_out * items[i].halves, 4);
  }
  return dtype == PNFX_F32 ? launch<pad_kernel<float>>(g.first[n], 256, 0, g, st, "pad")
                           : launch<pad_kernel<bf16>>(g.first[n], 256, 0, g, st, "pad");
}

}  // namespace pnfx
