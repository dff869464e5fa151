// Plain matrix products, the sum of their splits, and zero-padded copies.  What bounds the products and how they
// are staged: gemm.h.
#include <algorithm>
#include <cmath>

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

// The first `n` of eight elements (eight, where there are more).
template <typename T>
__device__ __forceinline__ void store_upto8(T* p, int n, const float* v) {
  if (n >= 8) return store8(p, v);
#pragma unroll
  for (int r = 0; r < 7; ++r)
    if (r < n) p[r] = from_f32<T>(v[r]);
}
__device__ __forceinline__ void load8(const float* p, int n, float* v) {
  typedef f32x4 V __attribute__((aligned(4)));
  if (n >= 8) {
    const f32x4 x = *reinterpret_cast<const V*>(p), y = *reinterpret_cast<const V*>(p + 4);
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = x[r], v[r + 4] = y[r];
    return;
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) v[r] = r < n ? p[r] : 0.f;
}

// Workgroup `block` of a product.
template <typename T, Kind KA, Kind KB, class C>
__device__ __forceinline__ void mm_tile(const MmArgs& g, int block, char* sm) {
  typedef Product<T, KA, KB, C> P;
  const int M = g.m_count ? min(g.M, *g.m_count) : g.M;
  const int tms = (M + C::TM - 1) / C::TM, tiles = tms * g.tn;
  if (block >= tiles * g.splits) return;
  // split by split: the tiles of one read the same k, and an XCD's workgroups are of few splits
  const int place = xcd_id(block, tiles * g.splits), split = place / tiles;
  int tm, tn;
  band_tile(place % tiles, tms, g.tn, tm, tn);
  const int m0 = tm * C::TM, n0 = tn * C::TN;
  const int K = g.k_count ? min((int)g.K, *g.k_count) : (int)g.K;
  const int all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  constexpr int WAVES = C::WM * C::WN;
  const int group = all / WAVES, wave = all % WAVES;
  int64_t k0 = split * g.steps * k_step<T>;
  const int64_t left = K - k0, most = g.steps * k_step<T>;
  int ks = (int)(left < most ? left : most);
  int steps = (ks + k_step<T> - 1) / k_step<T>;
  if constexpr (C::KG == 2) {  // as many steps for either group; past the end they read zeros
    steps = (steps + 1) / 2;
    const int half = steps * k_step<T>;
    k0 += group * half;
    ks = group ? ks - half : min(ks, half);
  }
  typename P::StageA sa;
  typename P::StageB sb;
  const T* a = static_cast<const T*>(g.a) + (KA == COL ? k0 * g.lda + m0 : m0 * g.lda + k0);
  const T* b = static_cast<const T*>(g.b) + (KB == COL ? k0 * g.ldb + n0 : n0 * g.ldb + k0);
  sa.init(a, g.lda, M - m0, ks, threadIdx.x % P::NT);
  sb.init(b, g.ldb, g.N - n0, ks, threadIdx.x % P::NT);
  f32x4 acc[P::MI][P::NJ] = {};
  P::run(sa, sb, steps, reinterpret_cast<T*>(sm + group * (lds_of<C> / C::KG)), wave, lane, acc);
  int i0 = 0, i1 = P::MI;
  if constexpr (C::KG == 2) {
    // each group adds up and stores half of the tile: the other half's sums go to the other group
    constexpr int H = P::MI / 2;
    f32x4* other = reinterpret_cast<f32x4*>(sm + group * (lds_of<C> / 2)) + wave * (H * P::NJ * 64) + lane;
    const f32x4* mine = reinterpret_cast<f32x4*>(sm + (group ^ 1) * (lds_of<C> / 2)) + wave * (H * P::NJ * 64) + lane;
#pragma unroll
    for (int i = 0; i < H; ++i)
#pragma unroll
      for (int j = 0; j < P::NJ; ++j) other[(i * P::NJ + j) * 64] = group ? acc[i][j] : acc[H + i][j];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < H; ++i)
#pragma unroll
      for (int j = 0; j < P::NJ; ++j) {
        if (group) acc[H + i][j] += mine[(i * P::NJ + j) * 64];
        else acc[i][j] += mine[(i * P::NJ + j) * 64];
      }
    i0 = group * H, i1 = i0 + H;
  }
  const int wm = wave / C::WN * P::MI, wn = wave % C::WN * P::NJ;
  float* sums = g.sums ? g.sums + (int64_t)split * g.M * g.N : nullptr;
  const float alpha = g.alpha ? *g.alpha : 1.f;
#pragma unroll
  for (int i = 0; i < P::MI; ++i) {
    if (C::KG == 2 && (i < i0 || i >= i1)) continue;
    const int m = m0 + stage_row<KA>(wm + i, lane & 15);
    const int row = out_row(m, g.gap_at, g.gap);
#pragma unroll
    for (int j = 0; j < P::NJ; j += 2) {
      const int n = n0 + pair_col<KB>(wn + j, lane);
      float v[8];
      pair8<KB>(acc[i][j], acc[i][j + 1], v);
      if (m >= M || n >= g.N) continue;
      if (sums) {
        float* s = sums + (int64_t)m * g.N + n;
        if (g.add) {
          float old[8];
          load8(s, g.N - n, old);
#pragma unroll
          for (int r = 0; r < 8; ++r) v[r] += old[r];
        }
        store_upto8(s, g.N - n, v);
      } else if (row >= 0) {
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] *= alpha;
        store_upto8(static_cast<T*>(g.c) + row * g.ldc + n, g.N - n, v);
      }
    }
  }
}

template <typename T, Kind KA, Kind KB, class C>
__global__ __launch_bounds__(threads_of<C>, 2) void mm_kernel(MmArgs g) {
  extern __shared__ __align__(16) char sm[];
  mm_tile<T, KA, KB, C>(g, blockIdx.x, sm);
}
// The products of a backward pass in one launch, none of which fills the chip by itself: first workgroups of each.
struct GroupArgs {
  MmArgs rc, cc[2];  // ROW COL, then COL COL
  int first[2];      // workgroups, a multiple of eight each
};
template <typename T, class C>
__global__ __launch_bounds__(threads_of<C>, 2) void mm_group_kernel(GroupArgs g) {
  extern __shared__ __align__(16) char sm[];
  const int block = blockIdx.x;
  if (block < g.first[0]) return mm_tile<T, ROW, COL, C>(g.rc, block, sm);
  const bool last = block >= g.first[1];
  mm_tile<T, COL, COL, C>(g.cc[last], block - g.first[last], sm);
}

struct SumArgs {
  const float* sums;
  void* c;
  const float* alpha;
  int64_t MN, ldc;
  int M, N, groups, splits, gap_at, gap;  // groups: of eight columns, in a row
};
constexpr int kMaxGroup = 3;
struct SumsArgs {
  SumArgs item[kMaxGroup];
  int64_t first[kMaxGroup + 1];  // workgroups
  int n;
};
// C from the splits' sums, added in split order: eight columns per thread.
template <typename T>
__global__ __launch_bounds__(256) void mm_sum_kernel(SumsArgs all) {
  int i = 0;
  while (i + 1 < all.n && (int64_t)blockIdx.x >= all.first[i + 1]) ++i;
  const SumArgs& g = all.item[i];
  const int64_t id = (blockIdx.x - all.first[i]) * 256 + threadIdx.x;
  const int m = (int)(id / g.groups), n = (int)(id % g.groups) * 8;
  if (m >= g.M) return;
  const int row = out_row(m, g.gap_at, g.gap);
  if (row < 0) return;
  const float* s = g.sums + (int64_t)m * g.N + n;
  float v[8] = {};
#pragma unroll 4
  for (int p = 0; p < g.splits; ++p) {
    float x[8];
    load8(s + p * g.MN, g.N - n, x);
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r] += x[r];
  }
  const float alpha = g.alpha ? *g.alpha : 1.f;
#pragma unroll
  for (int r = 0; r < 8; ++r) v[r] *= alpha;
  store_upto8(static_cast<T*>(g.c) + row * g.ldc + n, g.N - n, v);
}

constexpr int kMaxPads = 4;
struct PadArgs {
  PadItem item[kMaxPads];
  int64_t first[kMaxPads + 1];  // workgroups
  int n;
};
// Eight columns per thread, read at any alignment.
template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(PadArgs g) {
  int i = 0;
  while (i + 1 < g.n && (int64_t)blockIdx.x >= g.first[i + 1]) ++i;
  const PadItem& p = g.item[i];
  const int64_t id = (blockIdx.x - g.first[i]) * 256 + threadIdx.x, groups = p.cols_out / 8;
  const int64_t r = id / groups, c = id % groups * 8;
  if (r >= p.rows_out * p.halves) return;
  const int64_t half = r / p.rows_out, in = r % p.rows_out;
  const T* src = static_cast<const T*>(p.src) + (half * p.rows + in) * p.ld + c;
  T v[8];
  if (in < p.rows && c + 8 <= p.cols) {
    __builtin_memcpy(v, src, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = in < p.rows && c + e < p.cols ? src[e] : (T)0.f;
  }
  __builtin_memcpy(__builtin_assume_aligned(static_cast<T*>(p.dst) + r * p.cols_out + c, 16), v, sizeof(v));
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

// What a cut is expected to take.  A tile's step takes, with one of its kind on every CU, the time of its products at
// the rate that gemm.h's figures give, or half a microsecond if the step's loads are not hidden by another
// workgroup's products; a split's fp32 sums are written, and read by another kernel.
struct Cost {
  double work = 0, longest = 0, last = 0, after = 0;  // us of all workgroups, of one, and behind them
  bool summed = false;
  void add(int kind, const Shape& s, int dtype, int64_t splits, int64_t per) {
    const int es = dtype == PNFX_F32 ? 4 : 2;
    const int64_t T = kind == Cut::BIG ? 256 : 128, n = ceil_div(s.M, T) * ceil_div(s.N, T) * splits;
    const double rate = dtype == PNFX_F32 ? 120e6 : kind == Cut::BIG ? 1300e6 : 1050e6;  // operations per us, 256 CUs
    const double step = 2.0 * T * T * (128 / es) / (rate / 256);  // of one tile that has the CU to itself
    const double one = kind == Cut::MID   ? per * std::max(2 * step, 0.45) + 1.5
                       : kind == Cut::DUO ? ceil_div(per, 2) * std::max(2 * step, 0.45) + 2.0
                                          : per * step + 3.0;
    work += n * one;
    last = one;
    longest = std::max(longest, one);
    const double sums_us = (double)splits * s.M * s.N * 4 / 4e6;
    if (splits > 1 || s.sums) after += sums_us;
    if (splits > 1 && !s.sums) after += sums_us, summed = true;
  }
  double us(int kind) const {
    // rounds of the last product's workgroups
    const int64_t places = kind == Cut::MID ? 512 : 256;
    const double run = std::ceil(work / (places * last) - 1e-6) * last;
    return std::max(run, longest) + after + (summed ? 4.0 : 0);
  }
};

void cut_group(const Shape* shapes, int n, int dtype, bool can_split, Cut* cuts) {
  const int ks = 128 / (dtype == PNFX_F32 ? 4 : 2);
  int64_t most = 1;
  for (int i = 0; i < n; ++i) most = std::max(most, ceil_div(shapes[i].K, ks));
  double best = 1e30;
  for (int kind = 0; kind < 3; ++kind) {
    if (kind == Cut::BIG && dtype == PNFX_F32) continue;
    if (kind == Cut::DUO && !can_split) continue;
    // workgroups of all of k, and of half, a quarter, ... of the longest k, each about as long as the others
    for (int64_t len = most; len >= 4 || len == most; len = (len + 1) / 2) {
      Cut got[3];
      Cost cost;
      for (int i = 0; i < n; ++i) {
        const int64_t steps = std::max<int64_t>(1, ceil_div(shapes[i].K, ks));
        const int64_t splits = std::min<int64_t>(ceil_div(steps, len), 64), per = ceil_div(steps, splits);
        got[i] = Cut{(Cut::Kind)kind, (int)ceil_div(steps, per), per};
        cost.add(kind, shapes[i], dtype, got[i].splits, per);
      }
      const double us = cost.us(kind);
      if (us < best) {
        best = us;
        for (int i = 0; i < n; ++i) cuts[i] = got[i];
      }
      if (!can_split || len == 1) break;
    }
  }
}
Cut cut_of(int64_t M, int64_t N, int64_t K, int dtype, bool can_split) {
  const Shape s{M, N, K, false};
  Cut c;
  cut_group(&s, 1, dtype, can_split, &c);
  return c;
}

int64_t product_workspace(const Cut& cut, int64_t M, int64_t N) {
  return cut.splits > 1 ? cut.splits * M * N * 4 : 0;
}

// The kernel's arguments of a product; `ws`: where its splits' sums go, if it has any.
static int mm_args(const ProductArgs& p, const Cut& cut, int es, void* ws, MmArgs& g) {
  PNFX_REQUIRE(operand_ok(p.a, p.lda, es) && operand_ok(p.b, p.ldb, es), "product: operand alignment");
  PNFX_REQUIRE(p.M < (1 << 30) && p.N < (1 << 30) && p.K < (1 << 30), "product: %lld x %lld over %lld",
               (long long)p.M, (long long)p.N, (long long)p.K);
  const bool summed = !p.sums && cut.splits > 1;
  PNFX_REQUIRE(!summed || ws, "product: no workspace");
  const int64_t T = cut.kind == Cut::BIG ? 256 : 128;
  g.a = p.a;
  g.b = p.b;
  g.c = p.c;
  g.sums = summed ? static_cast<float*>(ws) : p.sums;
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
  return PNFX_OK;
}

static int sum_up(const Job* jobs, const MmArgs* g, int n, int dtype, hipStream_t st) {
  SumsArgs s;
  s.n = 0;
  s.first[0] = 0;
  for (int i = 0; i < n; ++i) {
    const ProductArgs& p = jobs[i].p;
    if (p.M < 1 || p.N < 1 || p.sums || jobs[i].cut.splits == 1) continue;
    const int64_t groups = ceil_div(p.N, 8);
    s.item[s.n] = SumArgs{g[i].sums, p.c, p.alpha, p.M * p.N, p.ldc, g[i].M, g[i].N, (int)groups, jobs[i].cut.splits,
                          g[i].gap_at, g[i].gap};
    s.first[s.n + 1] = s.first[s.n] + ceil_div(p.M * groups, 256);
    ++s.n;
  }
  if (!s.n) return PNFX_OK;
  return dtype == PNFX_F32 ? launch<mm_sum_kernel<float>>(s.first[s.n], 256, 0, s, st, "product sums")
                           : launch<mm_sum_kernel<bf16>>(s.first[s.n], 256, 0, s, st, "product sums");
}

int sum_splits(const float* sums, int splits, int64_t M, int64_t N, void* c, const float* alpha, int dtype,
               hipStream_t st) {
  const int64_t groups = ceil_div(N, 8);
  SumsArgs s;
  s.n = 1;
  s.item[0] = SumArgs{sums, c, alpha, M * N, N, (int)M, (int)N, (int)groups, splits, (int)M, 0};
  s.first[0] = 0;
  s.first[1] = ceil_div(M * groups, 256);
  return dtype == PNFX_F32 ? launch<mm_sum_kernel<float>>(s.first[1], 256, 0, s, st, "sum of splits")
                           : launch<mm_sum_kernel<bf16>>(s.first[1], 256, 0, s, st, "sum of splits");
}

template <typename T, class C>
static int group_launch(const GroupArgs& g, int64_t grid, hipStream_t st) {
  return launch<mm_group_kernel<T, C>>(grid, threads_of<C>, lds_of<C>, g, st, "products");
}

int products(const Job* jobs, int n, int dtype, hipStream_t st) {
  const int es = dtype == PNFX_F32 ? 4 : 2;
  PNFX_REQUIRE(n >= 1 && n <= kMaxGroup, "products: %d", n);
  MmArgs g[kMaxGroup] = {};
  bool group = n > 1 && jobs[0].ka == ROW && jobs[0].kb == COL;
  for (int i = 0; i < n; ++i) {
    PNFX_TRY(mm_args(jobs[i].p, jobs[i].cut, es, jobs[i].ws, g[i]));
    group = group && jobs[i].cut.kind == jobs[0].cut.kind && (i == 0 || (jobs[i].ka == COL && jobs[i].kb == COL));
  }
  if (group) {
    GroupArgs a = {};
    a.rc = g[0];
    a.cc[0] = g[1];
    a.cc[1] = g[n - 1];
    int64_t grid = 0;
    for (int i = 0; i < n; ++i) {
      // a multiple of eight: workgroup id % 8 is the XCD for every product (those left over end at once)
      grid += round_up((int64_t)g[i].tm * g[i].tn * g[i].splits, 8);
      PNFX_REQUIRE(grid < (1ll << 31), "products: %lld workgroups", (long long)grid);
      if (i < 2) a.first[i] = (int)grid;
    }
    const Cut::Kind kind = jobs[0].cut.kind;
    if (dtype == PNFX_F32)
      PNFX_TRY((kind == Cut::DUO ? group_launch<float, Duo>(a, grid, st) : group_launch<float, Mid>(a, grid, st)));
    else
      PNFX_TRY((kind == Cut::BIG   ? group_launch<bf16, Big>(a, grid, st)
                : kind == Cut::DUO ? group_launch<bf16, Duo>(a, grid, st)
                                   : group_launch<bf16, Mid>(a, grid, st)));
  } else {
    for (int i = 0; i < n; ++i) {
      const Job& j = jobs[i];
      if (dtype == PNFX_F32)
        PNFX_TRY((j.cut.kind == Cut::DUO ? mm_kinds<float, Duo>(j.ka, j.kb, g[i], st)
                                         : mm_kinds<float, Mid>(j.ka, j.kb, g[i], st)));
      else
        PNFX_TRY((j.cut.kind == Cut::BIG   ? mm_kinds<bf16, Big>(j.ka, j.kb, g[i], st)
                  : j.cut.kind == Cut::DUO ? mm_kinds<bf16, Duo>(j.ka, j.kb, g[i], st)
                                           : mm_kinds<bf16, Mid>(j.ka, j.kb, g[i], st)));
    }
  }
  return sum_up(jobs, g, n, dtype, st);
}

int pad(const PadItem* items, int n, int dtype, hipStream_t st) {
  if (!n) return PNFX_OK;
  PadArgs g;
  g.n = n;
  g.first[0] = 0;
  for (int i = 0; i < n; ++i) {
    g.item[i] = items[i];
    g.first[i + 1] = g.first[i] + ceil_div(items[i].rows_out * items[i].halves * (items[i].cols_out / 8), 256);
  }
  return dtype == PNFX_F32 ? launch<pad_kernel<float>>(g.first[n], 256, 0, g, st, "pad")
                           : launch<pad_kernel<bf16>>(g.first[n], 256, 0, g, st, "pad");
}

}  // namespace pnfx
