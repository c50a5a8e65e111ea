// Arguments of the 16-bit product core (gemm16.hip), shared with its callers.
#pragma once
#include "common.h"
#include "epilogue.h"

namespace rtat_native {

// D = epilogue(op(A) * op(B)) for `batch` matrices, A and B of `type` (F16 / BF16).
// tri == 1: the product is symmetric (m == n, no bias or aux, C symmetric): only tiles on or
// below the diagonal are computed and the others are written as their mirror images.
struct Gemm16 {
  int type;
  bool ta, tb;
  int m, n, k, batch, tri;
  const void* A;
  long lda, a_stride;
  const void* B;
  long ldb, b_stride;
  // 1: memory behind the operand's last column may be read up to a multiple of 8 rows.
  int a_roomy, b_roomy;
  // Bytes at the front of the handle's scratch that the caller uses for this product.
  size_t scratch_used;
  Epilogue ep;
};

rtat_status_t launch_gemm16(rtat_native_handle* h, const Gemm16& g);

// Rows of partial sums a gradient product of n columns leaves (Epilogue::sums), at most; and
// the kernel that adds `parts` rows of them, m long, in order.
int dact_sum_rows(int n);
rtat_status_t launch_sum_rows(rtat_native_handle* h, const float* parts, int count, int m,
                              float* out);

rtat_status_t launch_newton_schulz(rtat_native_handle* h, int g_type, int m, int n, int batch,
                                   const void* G, long ldg, long stride_g, int steps,
                                   const float* coeffs, float eps, void* O, long ldo,
                                   long stride_o);
size_t newton_schulz_workspace_bytes(int m, int n, int batch);

// dZ = dD * act'(Z) (skipped when dZ is null) and out[row] = sum over columns (skipped when null).
rtat_status_t launch_act_backward(rtat_native_handle* h, int type, int act, int m, int n,
                                  const void* dD, long lddd, const void* Z, long ldz, void* dZ,
                                  long lddz, float* dbias);
size_t dbias_workspace_bytes(int m, int n);
// The partial row sums' place in the handle's scratch, aligned; null when it cannot be had.
float* acquire_sums(rtat_native_handle* h, int m, int n);

}  // namespace rtat_native
