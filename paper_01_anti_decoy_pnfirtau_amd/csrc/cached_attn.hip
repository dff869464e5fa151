// The entry points of attention over the 8-bit cache: arguments, and how a call is cut.  The kernels are in
// cached_attn.h, built by head size in cached_attn_*.hip.
#include "cached_attn.h"

namespace pnfx {
namespace {

AttnPlan plan_of(int64_t B, int64_t H, int64_t G, int64_t N, int D, int64_t capacity, int bytes) {
  AttnPlan p = {};
  const int64_t rows = G * N;
  const int64_t tiles = (capacity + TILE - 1) / TILE, tall = B * H * ((rows + 127) / 128);
  // Waves that share their keys gain where turning these to bf16 is much of the work, heads of more than 64 columns, and
  // where there are workgroups of 128 rows for the whole card.  bf16, in us, shared and not:
  //   512 query tokens behind 7680, 2 sequences of 16 heads of 128: 131, 174; 4 of 16 heads of 64: 153, 136
  //   80 query tokens behind 7680, one sequence of 16 heads of 128: 42, 35
  //   prompts of 512 tokens, 16 of 8 heads of 128: 61, 113; 64 of 4 heads of 64: 61, 78; 16 of these: 24, 24; 8: 23, 14
  //   256 query tokens behind 256, 16 sequences of 8 heads of 128: 49, 64; 8 of these: 47, 35
  p.shared = bytes == 2 && D <= 128 && rows >= 256 && (tiles > 8 ? D > 64 : tall >= (D > 64 ? 256 : 512));
  p.NT = p.shared ? 2 : rows <= 16 || D > 128 ? 1 : 2;
  p.R = (int)((rows + 16 * p.NT - 1) / (16 * p.NT));
  const int waves = p.shared ? 4 : 1;  // of a unit that is cut
  p.R = (p.R + waves - 1) / waves * waves;
  p.units = B * H * p.R / waves;
  p.slots = p.shared ? 256 * RESIDENT_SHARED : 1024 * resident(bytes, D, p.NT);
  p.slot_rows = (int)std::min<int64_t>(rows, 16 * p.NT);
  // One workgroup a unit where no cut can gain: short caches, whose few tiles cost less than the join's launch (in us, whole and
  // cut, heads of 64: one token of 4 heads behind 1023 11.3, 14.5, behind 2047 12.5, 14.8; 100 tokens of 8 heads, 4
  // sequences behind 900 15, 20; 2048 tokens of 16 heads 127, 113), and enough units for the card to even out by itself
  // (one token, 16 heads, behind up to 1500, 800 sequences 239, 251; 64 tokens, 200 sequences 209, 169).
  if (tiles * std::max(D, 64) <= (p.R == 1 ? 2048 : 1024) || p.units >= (p.shared ? 2 : 4) * (int64_t)p.slots) return p;
  p.items = (std::min(p.units * tiles, p.units + p.slots) + 7) / 8 * 8 * waves;
  const auto round = [](int64_t x) { return (x + 255) & ~(int64_t)255; };
  // a wave for half of 1024 results, as a unit has at least two pieces, four a lane: 7.9 us for 4 sequences of 512 query
  // tokens behind up to 7680, 16 heads of 64; with twice as many waves 8.9
  p.join_waves = std::min(4, (p.slot_rows * D + 1023) / 1024);
  p.header_bytes = 256 + round(p.items * (int64_t)sizeof(Header));
  p.acc_bytes = round(p.items * p.slot_rows * D * 4);
  p.stat_bytes = round(p.items * 3 * p.slot_rows * 4);
  return p;
}

int run_any(const AttnArgs& a, const AttnPlan& p, int dtype, hipStream_t st) {
  if (dtype == PNFX_F32)
    return a.c.D <= 64 ? attn_f32_64(a, p, st) : a.c.D <= 128 ? attn_f32_128(a, p, st) : attn_f32_256(a, p, st);
  return a.c.D <= 64 ? attn_bf16_64(a, p, st) : a.c.D <= 128 ? attn_bf16_128(a, p, st) : attn_bf16_256(a, p, st);
}

}  // namespace
}  // namespace pnfx

extern "C" int64_t pnfx_cached_attn_workspace_size(const pnfx_cache* cache, int64_t Hq, int64_t N, int dtype) {
  using namespace pnfx;
  Cache c;
  if (cache_of(cache, "cached_attn", &c) || N < 1 || Hq < c.H || Hq % c.H) return 0;
  return plan_of(c.B, c.H, Hq / c.H, N, c.D, c.capacity(), dtype == PNFX_F32 ? 4 : 2).bytes();
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
  PNFX_REQUIRE(N >= 1 && Hq / a.c.H * N < (1ll << 31) - 256, "cached_attn: N=%lld", (long long)N);
  PNFX_REQUIRE(start || (start_all >= 0 && start_all < (1ll << 31)), "cached_attn: start %lld", (long long)start_all);
  const AttnPlan p = plan_of(a.c.B, a.c.H, Hq / a.c.H, N, a.c.D, a.c.capacity(), dtype == PNFX_F32 ? 4 : 2);
  PNFX_REQUIRE(p.units < (1ll << 24), "cached_attn: %lld row tiles in one call", (long long)p.units);
  PNFX_REQUIRE(!p.bytes() || (workspace && workspace_bytes >= p.bytes() &&
                              (reinterpret_cast<uintptr_t>(workspace) & 15) == 0),
               "cached_attn: workspace needs %lld bytes, 16-byte aligned", (long long)p.bytes());
  a.span = Span{start, counts, (int)start_all, (int)N};
  a.q = q, a.o = o, a.qsb = qsb, a.qsh = qsh, a.qsn = qsn, a.osb = osb, a.osh = osh, a.osn = osn;
  const int64_t parts = dtype == PNFX_F32 ? 2 : 4;  // elements of 8 bytes
  a.vec = a.c.d % 8 == 0 && qsb % parts == 0 && qsh % parts == 0 && qsn % parts == 0 &&
          (reinterpret_cast<uintptr_t>(q) & 7) == 0;
  a.tau = tau, a.scale = scale, a.gamma = gamma, a.has_gamma = has_gamma, a.causal = causal;
  a.G = (int)Hq / a.c.H, a.R = p.R, a.slots = p.slots, a.slot_rows = p.slot_rows;
  a.most_items = (int)p.items, a.join_waves = p.join_waves;
  char* ws = static_cast<char*>(workspace);
  a.items = reinterpret_cast<int*>(ws);
  a.headers = reinterpret_cast<Header*>(ws + 256);
  a.acc = reinterpret_cast<float*>(ws + p.header_bytes);
  a.stats = reinterpret_cast<float*>(ws + p.header_bytes + p.acc_bytes);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return run_any(a, p, dtype, st);
}
