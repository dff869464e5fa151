// The matrix product C[m][n] = sum_k A(m, k) B(n, k) that the feed-forward and cross-entropy kernels are built
// on: operand staging, tile loop and the choice of tiles.  Each kernel adds its own epilogue on the fp32
// accumulators.
//
// Operands go from global memory straight to LDS (buffer loads with LDS as destination, whose bounds check
// supplies the zeros past an edge), two tiles of 128 bytes of k deep, and from there to registers as MFMA
// fragments one phase ahead of the products that use them.  The loads of the tile after next are issued in two
// parts, A's behind the step's only barrier and B's a phase later, so that they do not queue up in front of
// the fragments' reads: 8192^3 in bf16 877 -> 838 us.
//
// Measured on MI355X, bf16, 8192^3 with 256 x 256 tiles: both operands as rows of k 795-840 us (1310-1380
// TFLOP/s; the library's product 766 us), rows by columns 815 us (872), columns by columns 837 us (984).
// 128 x 128 tiles of four waves 990-1025 us (1075-1110 TFLOP/s), two of which share a CU.  Bound by the LDS,
// which has to supply 192 KB of fragments and take 64 KB of tiles for every 2048 cycles of products.
#pragma once

#include <atomic>
#include <type_traits>

#include "tiles_bf16.h"

namespace pnfx {
namespace {

// Wait until at most N of this wave's vector-memory operations (direct-to-LDS loads among them) and no
// LDS operation are outstanding.
template <int N>
__device__ __forceinline__ void wait_vm_lgkm() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x70);
}

// A buffer descriptor over `bytes` bytes from p (both wave-uniform): loads past its end return zero.
__device__ __forceinline__ u32x4 buffer_of(const void* p, unsigned bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  u32x4 d;
  d[0] = __builtin_amdgcn_readfirstlane((unsigned)a);
  d[1] = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32) & 0xffff);
  d[2] = __builtin_amdgcn_readfirstlane(bytes);
  d[3] = 0x00027000;
  return d;
}
// 16 bytes per lane from buffer d at byte offset `off` to LDS bytes `lds` + 16 * lane.  In inline assembly:
// the compiler cannot tell the two LDS buffers of a pipelined loop apart and would wait for every such
// load before the next LDS read.  It has no output register; Product::run waits for the loads itself.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved: named all the same, as it is written
__device__ __forceinline__ void lds_dma16(u32x4 d, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(lds), "v"(off), "s"(d)
               : "m0", "memory");
}
#pragma clang diagnostic pop
__device__ __forceinline__ unsigned lds_addr(const void* p) {
  return (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void*)p);
}

// Element types.  A step covers 128 bytes of k; a fragment is 16 bytes of k of one row.
template <typename T>
struct Elem;
template <>
struct Elem<bf16> {
  typedef bf16x8 Frag;
};
template <>
struct Elem<float> {
  typedef f32x4 Frag;
};
template <typename T>
constexpr int k_step = 128 / (int)sizeof(T);
template <typename T>
constexpr int per16 = 16 / (int)sizeof(T);  // elements in 16 bytes

// acc[r] += sum_k b(row 4 (lane / 16) + r, k) a(row lane % 16, k), in mma_parts<T> instructions.
template <typename T>
constexpr int mma_parts = sizeof(T) == 4 ? 4 : 1;
__device__ __forceinline__ f32x4 mma_part(bf16x8 b, bf16x8 a, f32x4 acc, int) { return mfma16x16x32(b, a, acc); }
__device__ __forceinline__ f32x4 mma_part(f32x4 b, f32x4 a, f32x4 acc, int t) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(b[t], a[t], acc, 0, 0, 0);
}
template <typename F>
__device__ __forceinline__ f32x4 mma(F b, F a, f32x4 acc) {
#pragma unroll
  for (int t = 0; t < (sizeof(a[0]) == 4 ? 4 : 1); ++t) acc = mma_part(b, a, acc, t);
  return acc;
}

// Operands.  ROW: rows of k (element (r, k) at p[r ld + k]), staged as sub-tiles of 64 rows and read 16 bytes
// per lane.  COL: element (r, k) at p[k ld + r], staged as sub-tiles of 64 columns and read transposed.  PAIR:
// ROW from two matrices (the gate and the up projection), 32 rows of each in turn.
enum Kind { ROW, COL, PAIR };

// A sub-tile is 64 slots of 128 bytes; 16-byte chunk c of slot s lies at position c ^ stage_swz(s).  The
// swizzles depend on the slot's low four bits only, so that a fragment's block is a constant offset.  ROW: 16
// lanes read 16 consecutive slots at one chunk, which with two slots to the 64 banks lands on all of them.
// COL, bf16: a half wave reads 32 bytes, two chunks, of 8 consecutive slots: all banks too, with the same
// swizzle.  COL, fp32: a wave reads 64 bytes of 4 slots.
template <typename T, Kind KIND>
__device__ __forceinline__ int stage_swz(int slot) {
  if (KIND == COL && sizeof(T) == 4) return 4 * (slot >> 1 & 1);
  return (slot >> 1 & 3) << 1 | (slot >> 3 & 1);
}

// Stages tiles of R rows of one operand, NT threads, 16 bytes per thread and load.  Past `rows` and past K come
// zeros, or other elements of the same matrix where they only reach results that are not stored; past K
// zeros in both operands.  An operand's memory goes on to a whole 16-byte chunk of its inner dimension, which
// for ROW holds zeros there.
template <typename T, Kind KIND, int R, int NT>
struct Stage {
  static constexpr int NI = R * 8 / NT;  // loads per thread and step
  static constexpr int SPL = NT / 8;     // slots per load
  static_assert(SPL == 32 || SPL == 64, "a load fills half a sub-tile or a whole one");
  static constexpr int ES = (int)sizeof(T), KS = k_step<T>;
  const char* base[KIND == PAIR ? 2 : 1];  // element (first row, k0)
  int K, left;     // k of a tile, and those left of it
  int rows;        // rows from the tile's first on
  unsigned ldb;    // bytes from row to row
  unsigned limit;  // ROW, PAIR: bytes to the last row in reach; COL: bytes of a row in reach
  unsigned off;    // the lane's byte offset in load 0
  int ch;          // ROW: the lane's chunk of the step's k

  // p (PAIR: and p2): the tile's first row; nrows >= 1: how many there are from it on (PAIR: in each); k: its k.
  __device__ __forceinline__ void init(const T* p, int64_t ld, int nrows, int64_t k, int tid,
                                       const T* p2 = nullptr) {
    ldb = (unsigned)(ES * ld);
    K = left = (int)k;
    rows = nrows;
    base[0] = reinterpret_cast<const char*>(p);
    const int slot = tid / 8;
    ch = (tid % 8) ^ stage_swz<T, KIND>(slot);
    if constexpr (KIND == PAIR) base[1] = reinterpret_cast<const char*>(p2);
    if constexpr (KIND == COL) {
      limit = (unsigned)(ES * min(rows, R) + 15) & ~15u;
      // fp32: slot 32 h + 16 f + 4 t + g holds k = 16 f + 4 g + t of columns 32 h .. 32 h + 31
      const int k = ES == 4 ? (slot & 16) + 4 * (slot & 3) + (slot >> 2 & 3) : row_of_slot(slot);
      off = k * ldb + 16 * ch + (ES == 4 ? (slot >> 5) * 128 : 0);
    } else {
      const int row = row_of_slot(slot);
      set_limit();
      off = (KIND == PAIR ? row & 31 : row) * ldb + 16 * ch;
    }
  }
  __device__ __forceinline__ void set_limit() {
    limit = (unsigned)(min(rows, KIND == PAIR ? R / 2 : R) - 1) * ldb;
  }
  // ROW: the next steps are of the tile `by` rows further on, from its first k.
  __device__ __forceinline__ void move(int by, int steps) {
    static_assert(KIND == ROW, "");
    base[0] += (int64_t)by * ldb - 128 * steps;
    left = K;
    rows -= by;
    if (by) set_limit();
  }
  // The next step's tile to LDS byte address lds.
  __device__ __forceinline__ void load(unsigned lds, int wave) {
    // (in 32 bits: HIP's min and max of 64-bit integers go through double, 2 % of the large products' time)
    const unsigned ks = (unsigned)max(0, min(left, KS));
    const unsigned dst = lds + wave * 1024;
    if constexpr (KIND == COL) {
      const u32x4 d = buffer_of(base[0], ks ? (ks - 1) * ldb + limit : 0u);
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const unsigned o = ES == 4 ? j * SPL * 4
                                   : SPL == 64 ? 128 * j : (j & 1) * 32 * ldb + 128 * (j >> 1);
        lds_dma16(d, off + o, dst + j * NT * 16);
      }
      base[0] += (int64_t)KS * ldb;
    } else {
      // lanes past K read far out of the buffer
      const unsigned o0 = (unsigned)(per16<T> * ch) < ks ? off : 0x80000000u;
      const unsigned bytes = ks ? limit + ((ES * ks + 15) & ~15u) : 0u;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        if constexpr (KIND == PAIR) {
          const int half = SPL == 64 ? wave >> 2 : j & 1, g = SPL == 64 ? j : j >> 1;
          lds_dma16(buffer_of(half ? base[1] : base[0], bytes), o0 + g * 32 * ldb, dst + j * NT * 16);
        } else {
          lds_dma16(buffer_of(base[0], bytes), o0 + j * SPL * ldb, dst + j * NT * 16);
        }
      }
      base[0] += 128;
      if constexpr (KIND == PAIR) base[1] += 128;
    }
    left -= KS;
  }
};

// Fragments of a staged tile, in two halves of a step's k: lane group g of half hf holds, in bf16, k = 32 hf +
// 8 g + 0..7 and, in fp32, k = 16 hf + 4 g + 0..3.
template <typename T, Kind KIND>
struct Frags {
  typedef typename Elem<T>::Frag F;
  static constexpr int SUB = 64 * 128 / (int)sizeof(T);  // elements of a sub-tile
  const T* p[KIND == COL && sizeof(T) == 2 ? 4 : 2];
  // tile: the wave's first sub-tile in buffer 0
  __device__ __forceinline__ Frags(const T* tile, int lane) {
    const int r16 = lane & 15, g = lane >> 4;
    if constexpr (KIND == COL && sizeof(T) == 4) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
        p[b] = tile + g * 32 + 4 * ((4 * b + (r16 >> 2)) ^ stage_swz<T, COL>(g)) + (r16 & 3);
    } else if constexpr (KIND == COL) {
      const int e = (lane >> 2) & 3, q = lane & 3, sl = 4 * g + e;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        p[b] = tile + sl * 64 + 8 * ((2 * b + (q >> 1)) ^ stage_swz<T, COL>(sl)) + 4 * (q & 1);
    } else {
      constexpr int C = per16<T>;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
        p[hf] = tile + r16 * 8 * C + C * ((g + 4 * hf) ^ stage_swz<T, ROW>(r16));
    }
  }
  // 16-row block blk of the wave, `at` elements further on.
  __device__ __forceinline__ F get(int blk, int hf, int at) const {
    if constexpr (KIND == COL && sizeof(T) == 4) {
      const T* t = p[blk & 1] + at + (blk >> 2) * SUB + (blk >> 1 & 1) * (SUB / 2) + 16 * hf * 32;
      return F{t[0], t[4 * 32], t[8 * 32], t[12 * 32]};
    } else if constexpr (KIND == COL) {
      const T* t = p[blk & 3] + at + (blk >> 2) * SUB + 32 * hf * 64;
      return __builtin_shufflevector(ld_tr(t), ld_tr(t + 16 * 64), 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      return *reinterpret_cast<const F*>(p[hf] + at + blk * (SUB / 4));
    }
  }
};
// Row of the tile that index r (0..15) of block blk is.  PAIR: of 64 such rows the first 32 are 32 rows of the
// first matrix, the others the same rows of the second.
template <Kind KIND>
__device__ __forceinline__ int stage_row(int blk, int r) {
  return KIND == COL ? 16 * blk + r : 64 * (blk >> 2) + perm_row(blk & 3, r);
}

// The eight consecutive columns that a lane holds of one row after pair8 of the sums of blocks blk and blk + 1 (blk
// even).  ROW: those that perm_row gives the two blocks.  COL: the first four of a block are exchanged with
// the neighbouring lane group's, so that even groups hold columns of the first block and odd ones of the second.
template <Kind KB>
__device__ __forceinline__ int pair_col(int blk, int lane) {
  const int a = lane >> 4;
  return KB == COL ? 16 * (blk + (a & 1)) + 8 * (a >> 1) : stage_row<ROW>(blk, 4 * a);
}
template <Kind KB>
__device__ __forceinline__ void pair8(const f32x4& x, const f32x4& y, float* v) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if constexpr (KB == COL) {
      const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x[r]), __float_as_uint(y[r]), false, false);
      v[r] = __uint_as_float(s[0]);
      v[r + 4] = __uint_as_float(s[1]);
    } else {
      v[r] = x[r];
      v[r + 4] = y[r];
    }
  }
}
// Eight values to memory that is aligned to an element: gfx950 takes 16 bytes at any address.
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v) {
  if constexpr (sizeof(T) == 2) {
    typedef bf16x8 V __attribute__((aligned(2)));
    *reinterpret_cast<V*>(p) = pack8(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
  } else {
    typedef f32x4 V __attribute__((aligned(4)));
    *reinterpret_cast<V*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<V*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
  }
}

// Tiles of TM x TN by WM x WN waves, KG such groups of waves with a share of k each.  Big for products with tiles
// enough for every CU, two waves per SIMD; Mid, two workgroups per CU, for the others and for fp32; Duo, a CU's two
// Mid workgroups on the two halves of one tile's k, where there are fewer tiles than places for them.
struct Big {
  static constexpr int TM = 256, TN = 256, WM = 2, WN = 4, KG = 1;
};
struct Mid {
  static constexpr int TM = 128, TN = 128, WM = 2, WN = 2, KG = 1;
};
struct Duo {
  static constexpr int TM = 128, TN = 128, WM = 2, WN = 2, KG = 2;
};
template <class C>
constexpr int threads_of = 64 * C::WM * C::WN * C::KG;
template <class C>
constexpr int lds_of = C::KG * 2 * (C::TM + C::TN) * 128;

// acc[i][j][r] of a wave (wm, wn): row m = stage_row<KA>(wm MI + i, lane % 16), column n =
// stage_row<KB>(wn NJ + j, 4 (lane / 16) + r) of the tile.
template <typename T, Kind KA, Kind KB, class C>
struct Product {
  static constexpr int TM = C::TM, TN = C::TN, NT = threads_of<C> / C::KG;  // of a group of waves
  static constexpr int MI = TM / C::WM / 16, NJ = TN / C::WN / 16;
  static_assert(MI % 4 == 0 && NJ % 4 == 0, "a wave's share is whole sub-tiles");
  typedef Stage<T, KA, TM, NT> StageA;
  typedef Stage<T, KB, TN, NT> StageB;
  typedef typename Elem<T>::Frag F;

  // sm: lds_of<C> bytes, free; every wave's reads of it are done when run returns (its writes too).
  __device__ __forceinline__ static void run(StageA& sa, StageB& sb, int steps, T* sm, int wave, int lane,
                                             f32x4 (&acc)[MI][NJ]) {
    loop<false>(sa, sb, steps, 1, sm, wave, lane, acc, [](int) {});
  }
  // `tiles` tiles of TN rows of B below each other against the same rows of A: done(t) is called with tile t's
  // sums in acc, while the first steps of the next tile are on their way.
  template <class Done>
  __device__ __forceinline__ static void run_tiles(StageA& sa, StageB& sb, int steps, int tiles, T* sm, int wave,
                                                   int lane, f32x4 (&acc)[MI][NJ], Done done) {
    loop<true>(sa, sb, steps, tiles, sm, wave, lane, acc, done);
  }

 private:
  template <bool MANY, class Done>
  __device__ __forceinline__ static void loop(StageA& sa, StageB& sb, int steps, int tiles, T* sm, int wave, int lane,
                                              f32x4 (&acc)[MI][NJ], Done done) {
    if (steps <= 0 || tiles <= 0) return;
    const int total = MANY ? steps * tiles : steps;
    // both buffers of A, then both of B: an operand's fragments are within the 64 KB of an LDS load's offset
    constexpr int SA = TM * k_step<T>, SB = TN * k_step<T>, ES = (int)sizeof(T);
    const unsigned la = __builtin_amdgcn_readfirstlane(lds_addr(sm));
    const auto load_a = [&](int b) {
      sa.load(la + ES * b * SA, wave);
      if constexpr (MANY)
        if (sa.left <= 0) sa.move(0, steps);
    };
    const auto load_b = [&](int b) {
      sb.load(la + ES * (2 * SA + b * SB), wave);
      if constexpr (MANY)
        if (sb.left <= 0) sb.move(TN, steps);
    };
    const Frags<T, KA> fa(sm + wave / C::WN * MI * 16 * k_step<T>, lane);
    const Frags<T, KB> fb(sm + 2 * SA + wave % C::WN * NJ * 16 * k_step<T>, lane);
    // Four phases per step, (k-half, half of the row blocks): while one phase's products run, the
    // fragments of the next are read.
    constexpr int MH = MI / 2;
    F a[2][MH], b[2][NJ];
    const auto read_a = [&](int buf, int hf, int ih) {
#pragma unroll
      for (int i = 0; i < MH; ++i) a[ih][i] = fa.get(ih * MH + i, hf, buf * SA);
    };
    const auto read_b = [&](int buf, int hf) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) b[hf][j] = fb.get(j, hf, buf * SB);
    };
    const auto products = [&](int hf, int ih) {
      // (fp32: four products for each element of the fragment, no two in a row on the same sums)
#pragma unroll
      for (int t = 0; t < mma_parts<T>; ++t)
#pragma unroll
        for (int i = 0; i < MH; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            acc[ih * MH + i][j] = mma_part(b[hf][j], a[ih][i], acc[ih * MH + i][j], t);
      __builtin_amdgcn_sched_barrier(0);
    };
    load_a(0);
    load_b(0);
    if (total > 1) {
      load_a(1);
      load_b(1);
      wait_vm_lgkm<StageA::NI + StageB::NI>();
    } else {
      wait_vm_lgkm<0>();
    }
    __builtin_amdgcn_s_barrier();
    read_b(0, 0);
    read_a(0, 0, 0);
    int k = 0, tile = 0;
    const auto step = [&](int s, int buf) {
      if (s && s + 1 < total) load_b(buf ^ 1);
      __builtin_amdgcn_sched_barrier(0);
      read_a(buf, 0, 1);
      products(0, 0);
      read_b(buf, 1);
      read_a(buf, 1, 0);
      products(0, 1);
      read_a(buf, 1, 1);
      products(1, 0);
      // the next tile is here, and every wave has read this one
      wait_vm_lgkm<0>();
      __builtin_amdgcn_s_barrier();
      if (s + 2 < total) load_a(buf);
      __builtin_amdgcn_sched_barrier(0);
      read_b(buf ^ 1, 0);
      read_a(buf ^ 1, 0, 0);
      products(1, 1);
      if constexpr (MANY) {
        if (++k == steps) {
          done(tile++);
          k = 0;
#pragma unroll
          for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{};
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    int s = 0;
    for (; s + 1 < total; s += 2) {
      step(s, 0);
      step(s + 1, 1);
    }
    if (s < total) step(s, 0);
    wait_vm_lgkm<0>();
    __builtin_amdgcn_s_barrier();
  }
};

// Product::run_tiles for at most KS <= 4 steps of k: A's fragments stay in registers over all the tiles, which
// halves what the LDS has to supply (with 4 steps or fewer of products between two epilogues a tile's loop
// is otherwise bound by it), and B's steps go through a ring of four buffers, three of them ahead.  STORES: global
// stores that every done() issues (it may issue more); the loop does not wait for the latest ones.
template <typename T, int KS, class C, int STORES>
struct Thin {
  static constexpr int TM = C::TM, TN = C::TN, NT = threads_of<C>;
  static constexpr int MI = TM / C::WM / 16, NJ = TN / C::WN / 16;
  static constexpr int RING = 4;
  static constexpr int LDS = RING * TN * 128;
  static_assert(TM == TN, "A passes through the ring's buffers");
  typedef Stage<T, ROW, TM, NT> StageA;
  typedef Stage<T, ROW, TN, NT> StageB;
  typedef typename Elem<T>::Frag F;

  template <class Done>
  __device__ __forceinline__ static void run_tiles(StageA& sa, StageB& sb, int tiles, T* sm, int wave, int lane,
                                                   f32x4 (&acc)[MI][NJ], Done done) {
    if (tiles <= 0) return;
    constexpr int SB = TN * k_step<T>, ES = (int)sizeof(T);
    const unsigned la = __builtin_amdgcn_readfirstlane(lds_addr(sm));
    F a[KS][2][MI];
#pragma unroll
    for (int k = 0; k < KS; ++k) sa.load(la + ES * k * SB, wave);
    wait_vm_lgkm<0>();
    __builtin_amdgcn_s_barrier();
    const Frags<T, ROW> fa(sm + wave / C::WN * MI * 16 * k_step<T>, lane);
    const Frags<T, ROW> fb(sm + wave % C::WN * NJ * 16 * k_step<T>, lane);
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int i = 0; i < MI; ++i) a[k][hf][i] = fa.get(i, hf, k * SB);
    wait_vm_lgkm<0>();
    __builtin_amdgcn_s_barrier();
    const int total = KS * tiles;
    const auto load = [&](int s) {
      sb.load(la + ES * (s % RING) * SB, wave);
      if (sb.left <= 0) sb.move(TN, KS);
    };
    load(0);
    if (total > 1) load(1);
    if (total > 2) load(2);
    // Step s = KS t + k.  Its loads were issued in step s - 3, so that the loads of two steps may be outstanding
    // behind them, and the stores of the tiles that ended with step s - 3, s - 2 or s - 1 (from the fourth tile on).
    const auto step = [&](auto kc, int t) {
      constexpr int k = decltype(kc)::value;
      constexpr int ended = ((k + 2 * KS) % KS == 0) + ((k + 2 * KS - 1) % KS == 0) + ((k + 2 * KS - 2) % KS == 0);
      const int s = KS * t + k, buf = KS == RING ? k : s % RING;
      if (s + 2 >= total) wait_vm_lgkm<0>();
      else if (STORES && t >= 3) wait_vm_lgkm<2 * StageB::NI + STORES * ended>();
      else wait_vm_lgkm<2 * StageB::NI>();
      // and every wave has read step s - 1
      __builtin_amdgcn_s_barrier();
      if (s + 3 < total) load(s + 3);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        F b[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) b[j] = fb.get(j, hf, buf * SB);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[i][j] = mma(b[j], a[k][hf][i], k + hf ? acc[i][j] : f32x4{});
        if (KS == 4) __builtin_amdgcn_sched_barrier(0);  // no registers for both halves' fragments
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    for (int t = 0; t < tiles; ++t) {
      step(std::integral_constant<int, 0>{}, t);
      if constexpr (KS > 1) step(std::integral_constant<int, 1>{}, t);
      if constexpr (KS > 2) step(std::integral_constant<int, 2>{}, t);
      if constexpr (KS > 3) step(std::integral_constant<int, 3>{}, t);
      done(t);
      __builtin_amdgcn_sched_barrier(0);
    }
    wait_vm_lgkm<0>();
    __builtin_amdgcn_s_barrier();
  }
};

// Consecutive workgroups go to the eight XCDs in turn: the place of workgroup `id` of `total` in an order of which
// each XCD has a range of its own, so that its L2 holds what neighbours share.  (Where a number of rows is on the
// device, the total is of those, so that no XCD is left with workgroups that have nothing to do.)
__device__ __forceinline__ int xcd_id(int id, int total) {
  const int q = total / 8, r = total % 8, x = id % 8, y = id / 8;
  return x < r ? x * (q + 1) + y : r * (q + 1) + (x - r) * q + y;
}
// Tile `id` of tm x tn: column by column over bands of four tile rows.
__device__ __forceinline__ void band_tile(int id, int tm, int tn, int& m, int& n) {
  const int band = id / (4 * tn), first = 4 * band, high = min(tm - first, 4), in = id - band * 4 * tn;
  m = first + in % high;
  n = in / high;
}
__device__ __forceinline__ void tile_of(int id, int tm, int tn, int& m, int& n) {
  band_tile(xcd_id(id, tm * tn), tm, tn, m, n);
}

// Sizes that the staging's 32-bit byte offsets cover.
constexpr int64_t kMaxLd = 1 << 20;
inline bool operand_ok(const void* p, int64_t ld, int es) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * es % 16 == 0 && ld <= kMaxLd;
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// Launch with `lds` bytes of dynamic LDS; above 64 KB the kernel is told so, once on each device.
template <auto KERNEL, typename Arg>
int launch(int64_t grid, int threads, int lds, const Arg& a, hipStream_t st, const char* what) {
  if (grid <= 0) return PNFX_OK;
  // HIP counts a launch's threads in 32 bits
  PNFX_REQUIRE(grid * threads < (1ll << 32), "%s: %lld workgroups of %d", what, (long long)grid, threads);
  if (lds > 65536) {
    static std::atomic<uint64_t> told{0};
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (e == hipSuccess && !(told.load(std::memory_order_relaxed) & bit)) {
      e = hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL),
                              hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      told.fetch_or(bit, std::memory_order_relaxed);
    }
    if (e != hipSuccess) {
      set_error("%s: %s", what, hipGetErrorString(e));
      return PNFX_ELAUNCH;
    }
  }
  hipLaunchKernelGGL(KERNEL, dim3((unsigned)grid), dim3(threads), lds, st, a);
  return launch_status(what);
}

#define PNFX_TRY(call)             \
  do {                             \
    const int rc_ = (call);        \
    if (rc_ != PNFX_OK) return rc_; \
  } while (0)

}  // namespace
}  // namespace pnfx
