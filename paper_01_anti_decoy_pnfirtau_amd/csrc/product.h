// Products of two matrices with plain results, shared by the feed-forward and the cross-entropy entries
// (kernels in product.hip).
#pragma once

#include "gemm.h"

namespace pnfx {

// C[m][n] = sum_k A(m, k) B(n, k), M x N over K; A and B of one type, 16-byte aligned with rows in whole 16-byte
// chunks, ROW operands zero up to a whole chunk of k.  Only the combinations ROW ROW, ROW COL and COL COL.
struct ProductArgs {
  const void* a;
  const void* b;
  void* c;              // [*][ldc], the operands' type
  int64_t lda, ldb, ldc;
  int64_t M, N, K;
  // Rows of the product that are no rows of C: gap_at .. gap_at + gap - 1; those behind them move up.
  int64_t gap_at, gap;
  // Number of rows (m_count) or of k (k_count) in device memory, at most M or K; null: M, K.
  const int* m_count;
  const int* k_count;
  // Not null: fp32 sums [splits][M][N] instead of C, added to what is there (add) or written.
  float* sums;
  bool add;
  const float* alpha;  // one fp32 value in device memory that C is scaled by before it is rounded, or null
};

// How a product is cut: its tiles (gemm.h's Mid, Duo or Big) and the splits of its k over workgroups.
struct Cut {
  enum Kind { MID, DUO, BIG } kind;
  int splits;
  int64_t steps;  // steps of a split
  bool big() const { return kind == BIG; }
};
// can_split: whether k may be divided, over workgroups or a workgroup's waves.
Cut cut_of(int64_t M, int64_t N, int64_t K, int dtype, bool can_split);

// The cuts, of one kind, of up to three products that run in one launch.  sums: fp32 sums are wanted anyway.
struct Shape {
  int64_t M, N, K;
  bool sums;
};
void cut_group(const Shape* shapes, int n, int dtype, bool can_split, Cut* cuts);

// Workspace of a product with a C (not sums) at this cut, in bytes.
int64_t product_workspace(const Cut& cut, int64_t M, int64_t N);

// Up to three products that do not depend on each other: in one launch if the first is ROW COL, the others COL COL
// and their tiles of one kind.
struct Job {
  int ka, kb;  // operand kinds
  ProductArgs p;
  Cut cut;
  void* ws;
};
int products(const Job* jobs, int n, int dtype, hipStream_t stream);

// C [M][N] = alpha times the sum of `splits` fp32 matrices [M][N] in `sums`, in their order (alpha null: 1).
int sum_splits(const float* sums, int splits, int64_t M, int64_t N, void* c, const float* alpha, int dtype,
               hipStream_t stream);

// Copies of matrices with their columns zero-padded to whole 16-byte chunks, in one launch.
struct PadItem {
  const void* src;
  void* dst;         // [halves][rows_out][cols_out]
  int64_t ld;        // src elements from row to row
  int64_t rows, cols, rows_out, cols_out;
  int halves;        // matrices below each other in src
};
int pad(const PadItem* items, int n, int dtype, hipStream_t stream);

}  // namespace pnfx
