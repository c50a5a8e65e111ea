// extern "C" entry points of librtat_native (declared in include/rtat_native.h): argument
// checking, host-pointer scalars read by value, dispatch to the kernel launchers.
#include <new>
#include "common.h"
#include "gemm16.h"

#include <stdio.h>

#include <mutex>

using namespace rtat_native;

// Scratch of rtat_dtrsm_static: one array per GPU, part of the library's device image, held
// until the process ends.  Sized for a triangular matrix of order RTAT_DTRSM_STATIC_MAX_ORDER
// in either panel layout.  Host code never passes this name anywhere: it stands for the
// array only inside device code; the device address comes from hipGetSymbolAddress, once per
// device, in static_scratch_of below.
constexpr size_t scratch_bytes_for(int order) {
  const size_t tall = rtat_native::trsm_scratch_elems(order, rtat_native::PANEL_TALL, nullptr);
  const size_t low = rtat_native::trsm_scratch_elems(order, rtat_native::PANEL_SHORT, nullptr);
  return (tall > low ? tall : low) * sizeof(double) + 256;
}
constexpr size_t STATIC_SCRATCH_BYTES = scratch_bytes_for(RTAT_DTRSM_STATIC_MAX_ORDER);
static_assert(STATIC_SCRATCH_BYTES <= ((size_t)32 << 20), "the static scratch is meant to stay modest");
static __device__ __align__(256) unsigned char scratch[STATIC_SCRATCH_BYTES];

namespace rtat_native {

size_t trsm_workspace_bytes(int na);

// Device address of this device's copy of `scratch`, looked up the first time a handle is
// created on the device (with that device current) and remembered.  nullptr if the lookup
// failed.
static void* static_scratch_of(int device) {
  static std::mutex guard;
  static void* address[MAX_DEVICES] = {};
  static bool asked[MAX_DEVICES] = {};
  if (device < 0 || device >= MAX_DEVICES) return nullptr;
  std::lock_guard<std::mutex> lock(guard);
  if (!asked[device]) {
    int cur = -1;
    if (hipGetDevice(&cur) != hipSuccess || cur != device) {
      (void)hipGetLastError();
      return nullptr;  // only rtat_create asks first, and it asks for the current device
    }
    void* ptr = nullptr;
    if (hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch)) != hipSuccess) {
      (void)hipGetLastError();
      ptr = nullptr;
    }
    address[device] = ptr;
    asked[device] = true;
  }
  return address[device];
}

// Handle-owned scratch grows by allocating a new block (at least twice the old size, so the
// retired blocks of a handle never add up to more than its current one).  The old block is
// not freed here: kernels already enqueued, on this stream or on one the handle served
// before, and graphs captured earlier may still name it.  It is parked on the handle and
// freed by rtat_destroy.  Nothing synchronises.
void* acquire_workspace(rtat_native_handle* h, size_t bytes) {
  if (bytes == 0) return h->user_ws ? h->user_ws : h->own_ws;
  if (h->user_ws != nullptr) return h->user_ws_bytes >= bytes ? h->user_ws : nullptr;
  if (h->own_ws_bytes < bytes) {
    if (stream_capturing(h->stream)) return nullptr;
    size_t want = 2 * h->own_ws_bytes;
    if (want < bytes) want = bytes;
    void* p = nullptr;
    if (malloc_on_device(h->device, &p, want) != hipSuccess) {
      (void)hipGetLastError();
      want = bytes;
      if (malloc_on_device(h->device, &p, want) != hipSuccess) {
        (void)hipGetLastError();
        return nullptr;
      }
    }
    if (h->own_ws != nullptr) {
      try {
        h->retired_ws.push_back(h->own_ws);
      } catch (...) {  // no room to remember the old block: keep using it
        (void)hipFree(p);
        return nullptr;
      }
    }
    h->own_ws = p;
    h->own_ws_bytes = want;
  }
  return h->own_ws;
}

}  // namespace rtat_native

namespace {

// The handle's device made current for the length of a call.
struct OnDevice {
  int before = -1;
  explicit OnDevice(const rtat_native_handle* h) {
    if (hipGetDevice(&before) != hipSuccess) {
      (void)hipGetLastError();
      before = -1;
    }
    if (before == h->device) before = -1;
    else (void)hipSetDevice(h->device);
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

bool valid_half(int type) { return type == RTAT_TYPE_F16 || type == RTAT_TYPE_BF16; }
bool valid_act(int act) { return act >= 0 && act < RTAT_ACT_COUNT; }
bool short_ld(int ld, int rows) { return ld < (rows > 1 ? rows : 1); }
// A launch holds fewer than 2^32 threads: 2^30 rows in 64 x 64 tiles of 256 are one too many.
bool too_long(int m, int n, int k) {
  constexpr int most = (1 << 30) - 1024;
  return m > most || n > most || k > most;
}

// Shared checks of the 16-bit products: sizes, and the operands when they are read.
rtat_status_t check_product(int type, int transa, int transb, int m, int n, int k,
                            const float* alpha, const void* A, int lda, const void* B, int ldb) {
  if (!valid_half(type) || !valid_op(transa) || !valid_op(transb)) return RTAT_STATUS_INVALID_ENUM;
  if (m < 0 || n < 0 || k < 0 || alpha == nullptr) return RTAT_STATUS_INVALID_VALUE;
  if (too_long(m, n, k)) return RTAT_STATUS_NOT_SUPPORTED;
  if (m == 0 || n == 0 || k == 0 || *alpha == 0.0f) return RTAT_STATUS_SUCCESS;
  if (A == nullptr || B == nullptr || short_ld(lda, transa == RTAT_OP_T ? k : m) ||
      short_ld(ldb, transb == RTAT_OP_T ? n : k))
    return RTAT_STATUS_INVALID_VALUE;
  return RTAT_STATUS_SUCCESS;
}

Gemm16 product(int type, bool ta, bool tb, int m, int n, int k, float alpha, const void* A,
               long lda, const void* B, long ldb) {
  Gemm16 g = {};
  g.type = type;
  g.ta = ta;
  g.tb = tb;
  g.m = m;
  g.n = n;
  g.k = alpha == 0.0f ? 0 : k;
  g.batch = 1;
  g.A = A;
  g.lda = lda;
  g.B = B;
  g.ldb = ldb;
  g.ep.rows = m;
  g.ep.cols = n;
  g.ep.alpha = alpha;
  g.ep.bias_type = g.ep.aux_type = type;
  return g;
}

}  // namespace

#define RTAT_CHECK_HANDLE(h) \
  if ((h) == nullptr) return RTAT_STATUS_HANDLE_IS_NULLPTR

extern "C" {

rtat_status_t rtat_create(rtat_handle_t* handle) {
  if (handle == nullptr) return RTAT_STATUS_INVALID_VALUE;
  *handle = nullptr;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) {
    (void)hipGetLastError();
    return RTAT_STATUS_NOT_INITIALIZED;
  }
  hipDeviceProp_t prop;
  if (hipGetDeviceProperties(&prop, dev) != hipSuccess) {
    (void)hipGetLastError();
    return RTAT_STATUS_NOT_INITIALIZED;
  }
  rtat_native_handle* h = new (std::nothrow) rtat_native_handle();
  if (h == nullptr) return RTAT_STATUS_ALLOC_FAILED;
  h->device = dev;
  h->compute_units = prop.multiProcessorCount;
  h->clock_hz = (double)prop.clockRate * 1e3;
  h->mem_bytes_per_s = 2.0 * (double)prop.memoryClockRate * 1e3 * (double)prop.memoryBusWidth / 8.0;
  h->max_dyn_lds = prop.sharedMemPerBlock;
  // The scratch for GEMM / SYRK tail slices comes with the handle, so that no compute call
  // ever allocates it inside a caller's event pair.  Without it tails are computed unsplit.
  prepare_split_workspace(h);
  h->static_ws = static_scratch_of(dev);
  *handle = h;
  return RTAT_STATUS_SUCCESS;
}

rtat_status_t rtat_destroy(rtat_handle_t h) {
  RTAT_CHECK_HANDLE(h);
  if (h->own_ws != nullptr || h->split_ws != nullptr || !h->retired_ws.empty()) {
    // Freeing device memory while a stream records into a graph would invalidate the capture:
    // refuse, and leave the handle as it is.
    if (stream_capturing(h->stream)) return RTAT_STATUS_NOT_SUPPORTED;
    // Work still in flight on any stream of the handle's device may name the blocks: let that
    // device drain first, whichever device is current on this thread.
    int cur = -1;
    if (hipGetDevice(&cur) != hipSuccess) cur = -1;
    if (cur != h->device) (void)hipSetDevice(h->device);
    (void)hipDeviceSynchronize();
    if (h->own_ws != nullptr) (void)hipFree(h->own_ws);
    for (void* p : h->retired_ws) (void)hipFree(p);
    if (h->split_ws != nullptr) (void)hipFree(h->split_ws);
    if (cur != h->device && cur >= 0) (void)hipSetDevice(cur);
    (void)hipGetLastError();
  }
  delete h;
  return RTAT_STATUS_SUCCESS;
}

rtat_status_t rtat_set_stream(rtat_handle_t h, rtat_stream_t stream) {
  RTAT_CHECK_HANDLE(h);
  h->stream = static_cast<hipStream_t>(stream);
  return RTAT_STATUS_SUCCESS;
}

rtat_status_t rtat_get_stream(rtat_handle_t h, rtat_stream_t* stream) {
  RTAT_CHECK_HANDLE(h);
  if (stream == nullptr) return RTAT_STATUS_INVALID_VALUE;
  *stream = static_cast<rtat_stream_t>(h->stream);
  return RTAT_STATUS_SUCCESS;
}

rtat_status_t rtat_set_workspace(rtat_handle_t h, void* device_ptr, size_t bytes) {
  RTAT_CHECK_HANDLE(h);
  if ((device_ptr == nullptr) != (bytes == 0)) return RTAT_STATUS_INVALID_VALUE;
  h->user_ws = device_ptr;
  h->user_ws_bytes = bytes;
  return RTAT_STATUS_SUCCESS;
}

size_t rtat_dtrsm_workspace_bytes(rtat_side_t side, int m, int n) {
  return trsm_workspace_bytes(side == RTAT_SIDE_LEFT ? m : n);
}

rtat_status_t rtat_dgemm_ex(rtat_handle_t h, rtat_operation_t transa, rtat_operation_t transb,
                            int m, int n, int k, const double* alpha, const double* A, int lda,
                            const double* B, int ldb, const double* beta, double* C, int ldc,
                            int variant) {
  RTAT_CHECK_HANDLE(h);
  if (!valid_op(transa) || !valid_op(transb)) return RTAT_STATUS_INVALID_ENUM;
  if (alpha == nullptr || beta == nullptr) return RTAT_STATUS_INVALID_VALUE;
  return launch_dgemm(h, transa == RTAT_OP_T, transb == RTAT_OP_T, m, n, k, *alpha, A, lda, B,
                      ldb, *beta, C, ldc, 0, variant);
}

rtat_status_t rtat_dgemm(rtat_handle_t h, rtat_operation_t transa, rtat_operation_t transb,
                         int m, int n, int k, const double* alpha, const double* A, int lda,
                         const double* B, int ldb, const double* beta, double* C, int ldc) {
  return rtat_dgemm_ex(h, transa, transb, m, n, k, alpha, A, lda, B, ldb, beta, C, ldc,
                       RTAT_GEMM_AUTO);
}

rtat_status_t rtat_dsyrk_ex(rtat_handle_t h, rtat_fill_t uplo, rtat_operation_t trans, int n,
                            int k, const double* alpha, const double* A, int lda,
                            const double* beta, double* C, int ldc, int variant) {
  RTAT_CHECK_HANDLE(h);
  if (!valid_fill(uplo) || !valid_op(trans)) return RTAT_STATUS_INVALID_ENUM;
  if (alpha == nullptr || beta == nullptr) return RTAT_STATUS_INVALID_VALUE;
  // op(A) op(A)^T: trans == N -> A (n x k) times A^T; trans == T -> A^T times A (A is k x n).
  const bool t = trans == RTAT_OP_T;
  return launch_dgemm(h, t, !t, n, n, k, *alpha, A, lda, A, lda, *beta, C, ldc,
                      uplo == RTAT_FILL_LOWER ? 1 : 2, variant);
}

rtat_status_t rtat_dsyrk(rtat_handle_t h, rtat_fill_t uplo, rtat_operation_t trans, int n, int k,
                         const double* alpha, const double* A, int lda, const double* beta,
                         double* C, int ldc) {
  return rtat_dsyrk_ex(h, uplo, trans, n, k, alpha, A, lda, beta, C, ldc, RTAT_GEMM_AUTO);
}

rtat_status_t rtat_dtrsm_ex(rtat_handle_t h, rtat_side_t side, rtat_fill_t uplo,
                            rtat_operation_t trans, rtat_diag_t diag, int m, int n,
                            const double* alpha, const double* A, int lda, double* B, int ldb,
                            int variant) {
  RTAT_CHECK_HANDLE(h);
  if (!valid_side(side) || !valid_fill(uplo) || !valid_op(trans) || !valid_diag(diag))
    return RTAT_STATUS_INVALID_ENUM;
  if (alpha == nullptr) return RTAT_STATUS_INVALID_VALUE;
  return launch_trsm<double>(h, side == RTAT_SIDE_LEFT, uplo == RTAT_FILL_LOWER, trans == RTAT_OP_T,
                      diag == RTAT_DIAG_UNIT, m, n, *alpha, A, lda, B, ldb, variant);
}

rtat_status_t rtat_dtrsm(rtat_handle_t h, rtat_side_t side, rtat_fill_t uplo,
                         rtat_operation_t trans, rtat_diag_t diag, int m, int n,
                         const double* alpha, const double* A, int lda, double* B, int ldb) {
  return rtat_dtrsm_ex(h, side, uplo, trans, diag, m, n, alpha, A, lda, B, ldb, RTAT_GEMM_AUTO);
}

rtat_status_t rtat_dtrsm_static(rtat_handle_t h, rtat_side_t side, rtat_fill_t uplo,
                                rtat_operation_t trans, rtat_diag_t diag, int m, int n,
                                const double* alpha, const double* A, int lda, double* B,
                                int ldb) {
  RTAT_CHECK_HANDLE(h);
  if (!valid_side(side) || !valid_fill(uplo) || !valid_op(trans) || !valid_diag(diag))
    return RTAT_STATUS_INVALID_ENUM;
  if (alpha == nullptr) return RTAT_STATUS_INVALID_VALUE;
  const int na = side == RTAT_SIDE_LEFT ? m : n;
  if (na > RTAT_DTRSM_STATIC_MAX_ORDER) return RTAT_STATUS_NOT_SUPPORTED;
  if (h->static_ws == nullptr) return RTAT_STATUS_NOT_INITIALIZED;
  // The solve runs as it does with a lent workspace (no allocation anywhere below, GEMM
  // tails unsplit), the lent buffer being this device's static array.  Every element of
  // the scratch a solve reads, it has written first: nothing needs clearing between calls.
  void* const lent = h->user_ws;
  const size_t lent_bytes = h->user_ws_bytes;
  h->user_ws = h->static_ws;
  h->user_ws_bytes = STATIC_SCRATCH_BYTES;
  const rtat_status_t st =
      launch_trsm<double>(h, side == RTAT_SIDE_LEFT, uplo == RTAT_FILL_LOWER, trans == RTAT_OP_T,
                          diag == RTAT_DIAG_UNIT, m, n, *alpha, A, lda, B, ldb, RTAT_GEMM_AUTO);
  h->user_ws = lent;
  h->user_ws_bytes = lent_bytes;
  return st;
}

rtat_status_t rtat_dgeam(rtat_handle_t h, rtat_operation_t transa, rtat_operation_t transb,
                         int m, int n, const double* alpha, const double* A, int lda,
                         const double* beta, const double* B, int ldb, double* C, int ldc) {
  RTAT_CHECK_HANDLE(h);
  if (!valid_op(transa) || !valid_op(transb)) return RTAT_STATUS_INVALID_ENUM;
  if (alpha == nullptr || beta == nullptr) return RTAT_STATUS_INVALID_VALUE;
  return launch_geam<double>(h, transa == RTAT_OP_T, transb == RTAT_OP_T, m, n, *alpha, A, lda,
                             *beta, B, ldb, C, ldc);
}

rtat_status_t rtat_sgemm_ex(rtat_handle_t h, rtat_operation_t transa, rtat_operation_t transb,
                            int m, int n, int k, const float* alpha, const float* A, int lda,
                            const float* B, int ldb, const float* beta, float* C, int ldc,
                            int variant) {
  RTAT_CHECK_HANDLE(h);
  if (!valid_op(transa) || !valid_op(transb)) return RTAT_STATUS_INVALID_ENUM;
  if (alpha == nullptr || beta == nullptr) return RTAT_STATUS_INVALID_VALUE;
  return launch_gemm<float>(h, transa == RTAT_OP_T, transb == RTAT_OP_T, m, n, k, *alpha, A, lda,
                            B, ldb, *beta, C, ldc, 0, variant);
}

rtat_status_t rtat_sgemm(rtat_handle_t h, rtat_operation_t transa, rtat_operation_t transb,
                         int m, int n, int k, const float* alpha, const float* A, int lda,
                         const float* B, int ldb, const float* beta, float* C, int ldc) {
  return rtat_sgemm_ex(h, transa, transb, m, n, k, alpha, A, lda, B, ldb, beta, C, ldc,
                       RTAT_GEMM_AUTO);
}

rtat_status_t rtat_ssyrk_ex(rtat_handle_t h, rtat_fill_t uplo, rtat_operation_t trans, int n,
                            int k, const float* alpha, const float* A, int lda,
                            const float* beta, float* C, int ldc, int variant) {
  RTAT_CHECK_HANDLE(h);
  if (!valid_fill(uplo) || !valid_op(trans)) return RTAT_STATUS_INVALID_ENUM;
  if (alpha == nullptr || beta == nullptr) return RTAT_STATUS_INVALID_VALUE;
  const bool t = trans == RTAT_OP_T;
  return launch_gemm<float>(h, t, !t, n, n, k, *alpha, A, lda, A, lda, *beta, C, ldc,
                            uplo == RTAT_FILL_LOWER ? 1 : 2, variant);
}

rtat_status_t rtat_ssyrk(rtat_handle_t h, rtat_fill_t uplo, rtat_operation_t trans, int n, int k,
                         const float* alpha, const float* A, int lda, const float* beta,
                         float* C, int ldc) {
  return rtat_ssyrk_ex(h, uplo, trans, n, k, alpha, A, lda, beta, C, ldc, RTAT_GEMM_AUTO);
}

rtat_status_t rtat_strsm_ex(rtat_handle_t h, rtat_side_t side, rtat_fill_t uplo,
                            rtat_operation_t trans, rtat_diag_t diag, int m, int n,
                            const float* alpha, const float* A, int lda, float* B, int ldb,
                            int variant) {
  RTAT_CHECK_HANDLE(h);
  if (!valid_side(side) || !valid_fill(uplo) || !valid_op(trans) || !valid_diag(diag))
    return RTAT_STATUS_INVALID_ENUM;
  if (alpha == nullptr) return RTAT_STATUS_INVALID_VALUE;
  return launch_trsm<float>(h, side == RTAT_SIDE_LEFT, uplo == RTAT_FILL_LOWER,
                            trans == RTAT_OP_T, diag == RTAT_DIAG_UNIT, m, n, *alpha, A, lda, B,
                            ldb, variant);
}

rtat_status_t rtat_strsm(rtat_handle_t h, rtat_side_t side, rtat_fill_t uplo,
                         rtat_operation_t trans, rtat_diag_t diag, int m, int n,
                         const float* alpha, const float* A, int lda, float* B, int ldb) {
  return rtat_strsm_ex(h, side, uplo, trans, diag, m, n, alpha, A, lda, B, ldb, RTAT_GEMM_AUTO);
}

rtat_status_t rtat_sgeam(rtat_handle_t h, rtat_operation_t transa, rtat_operation_t transb,
                         int m, int n, const float* alpha, const float* A, int lda,
                         const float* beta, const float* B, int ldb, float* C, int ldc) {
  RTAT_CHECK_HANDLE(h);
  if (!valid_op(transa) || !valid_op(transb)) return RTAT_STATUS_INVALID_ENUM;
  if (alpha == nullptr || beta == nullptr) return RTAT_STATUS_INVALID_VALUE;
  return launch_geam<float>(h, transa == RTAT_OP_T, transb == RTAT_OP_T, m, n, *alpha, A, lda,
                            *beta, B, ldb, C, ldc);
}

const char* rtat_gemm_variant_name(int variant) {
  switch (variant) {
    case RTAT_GEMM_AUTO: return "auto";
    case RTAT_GEMM_T256x128: return "256x128";
    case RTAT_GEMM_T128x128: return "128x128";
    case RTAT_GEMM_T128x64: return "128x64";
    case RTAT_GEMM_T64x64: return "64x64";
    default: return nullptr;
  }
}

const char* rtat_tail_mode_name(int mode) {
  switch (mode) {
    case RTAT_TAIL_AUTO: return "auto";
    case RTAT_TAIL_WHOLE: return "whole";
    case RTAT_TAIL_SPLIT: return "split";
    default: return nullptr;
  }
}

const char* rtat_trsm_panel_name(int panel) {
  switch (panel) {
    case RTAT_PANEL_AUTO: return "auto";
    case RTAT_PANEL_512: return "512";
    case RTAT_PANEL_1024: return "1024";
    default: return nullptr;
  }
}

rtat_status_t rtat_last_launch(rtat_handle_t h, rtat_launch_info_t* info) {
  RTAT_CHECK_HANDLE(h);
  if (info == nullptr) return RTAT_STATUS_INVALID_VALUE;
  *info = h->last;
  if (h->last_bm > 0) snprintf(info->tile, sizeof(info->tile), "%dx%d", h->last_bm, h->last_bn);
  return RTAT_STATUS_SUCCESS;
}

rtat_status_t rtat_dfill(rtat_handle_t h, double* A, int m, int n, int ld, uint64_t seed,
                         int kind) {
  RTAT_CHECK_HANDLE(h);
  return launch_fill<double>(h, A, m, n, ld, seed, kind);
}

rtat_status_t rtat_sfill(rtat_handle_t h, float* A, int m, int n, int ld, uint64_t seed,
                         int kind) {
  RTAT_CHECK_HANDLE(h);
  return launch_fill<float>(h, A, m, n, ld, seed, kind);
}

rtat_status_t rtat_device_peaks(rtat_handle_t h, double* fp64_mfma_flops,
                                double* hbm_bytes_per_s, int* compute_units) {
  RTAT_CHECK_HANDLE(h);
  // 128 fp64 matrix flop per clock per CU on CDNA4 (v_mfma_f64_16x16x4: 2048 flop in 64
  // cycles on each of 4 SIMDs).
  if (fp64_mfma_flops) *fp64_mfma_flops = (double)h->compute_units * h->clock_hz * 128.0;
  if (hbm_bytes_per_s) *hbm_bytes_per_s = h->mem_bytes_per_s;
  if (compute_units) *compute_units = h->compute_units;
  return RTAT_STATUS_SUCCESS;
}

rtat_status_t rtat_dmove_pair(rtat_handle_t h, const rtat_move_t* first,
                              const rtat_move_t* second) {
  RTAT_CHECK_HANDLE(h);
  if (first == nullptr || second == nullptr) return RTAT_STATUS_INVALID_VALUE;
  return launch_move_pair<double>(h, first, second);
}

rtat_status_t rtat_smove_pair(rtat_handle_t h, const rtat_move_t* first,
                              const rtat_move_t* second) {
  RTAT_CHECK_HANDLE(h);
  if (first == nullptr || second == nullptr) return RTAT_STATUS_INVALID_VALUE;
  return launch_move_pair<float>(h, first, second);
}

rtat_status_t rtat_hbm_probe(rtat_handle_t h, int kind, const void* src, void* dst,
                             size_t bytes) {
  RTAT_CHECK_HANDLE(h);
  return launch_probe(h, kind, src, dst, bytes);
}

rtat_status_t rtat_gemm_ep(rtat_handle_t h, rtat_type_t type, rtat_operation_t transa,
                           rtat_operation_t transb, int m, int n, int k, const float* alpha,
                           const void* A, int lda, const void* B, int ldb,
                           const rtat_epilogue_t* ep, const float* beta, const void* C, int ldc,
                           rtat_type_t d_type, void* D, int ldd) {
  RTAT_CHECK_HANDLE(h);
  rtat_status_t st = check_product(type, transa, transb, m, n, k, alpha, A, lda, B, ldb);
  if (st != RTAT_STATUS_SUCCESS) return st;
  if ((d_type != type && d_type != RTAT_TYPE_F32) || (ep != nullptr && !valid_act(ep->act)))
    return RTAT_STATUS_INVALID_ENUM;
  if (beta == nullptr) return RTAT_STATUS_INVALID_VALUE;
  if (m == 0 || n == 0) return RTAT_STATUS_SUCCESS;
  if (D == nullptr || short_ld(ldd, m)) return RTAT_STATUS_INVALID_VALUE;
  if (*beta != 0.0f && (C == nullptr || short_ld(ldc, m))) return RTAT_STATUS_INVALID_VALUE;
  if (ep != nullptr && ep->aux != nullptr && short_ld(ep->ldaux, m)) return RTAT_STATUS_INVALID_VALUE;
  Gemm16 g = product(type, transa == RTAT_OP_T, transb == RTAT_OP_T, m, n, k, *alpha, A, lda, B, ldb);
  if (ep != nullptr) {
    g.ep.act = ep->act;
    g.ep.bias = ep->bias;
    g.ep.aux = ep->aux;
    g.ep.ldaux = ep->ldaux;
  }
  g.ep.beta = *beta;
  g.ep.C = *beta != 0.0f ? C : nullptr;
  g.ep.ldc = ldc;
  g.ep.c_type = g.ep.d_type = d_type;
  g.ep.D = D;
  g.ep.ldd = ldd;
  OnDevice on(h);
  return launch_gemm16(h, g);
}

rtat_status_t rtat_gemm_ep_backward(rtat_handle_t h, rtat_type_t type, rtat_operation_t transa,
                                    rtat_operation_t transb, int m, int n, int k,
                                    const float* alpha, const void* A, int lda, const void* B,
                                    int ldb, rtat_activation_t act, const void* Z, int ldz,
                                    const void* dD, int lddd, const rtat_gemm_grads_t* grads) {
  RTAT_CHECK_HANDLE(h);
  if (!valid_half(type) || !valid_op(transa) || !valid_op(transb) || !valid_act(act))
    return RTAT_STATUS_INVALID_ENUM;
  if (m < 0 || n < 0 || k < 0 || alpha == nullptr || grads == nullptr) return RTAT_STATUS_INVALID_VALUE;
  if (too_long(m, n, k)) return RTAT_STATUS_NOT_SUPPORTED;
  const rtat_gemm_grads_t& q = *grads;
  const bool ta = transa == RTAT_OP_T, tb = transb == RTAT_OP_T;
  const bool want_a = q.dA != nullptr && m > 0 && k > 0, want_b = q.dB != nullptr && n > 0 && k > 0;
  const bool slope = act != RTAT_ACT_NONE, some = m > 0 && n > 0;
  if ((q.dA != nullptr && q.da_type != type && q.da_type != RTAT_TYPE_F32) ||
      (q.dB != nullptr && q.db_type != type && q.db_type != RTAT_TYPE_F32))
    return RTAT_STATUS_INVALID_ENUM;
  if ((want_a && short_ld(q.ldda, ta ? k : m)) || (want_b && short_ld(q.lddb, tb ? n : k)))
    return RTAT_STATUS_INVALID_VALUE;
  if (some) {
    if (dD == nullptr || short_ld(lddd, m)) return RTAT_STATUS_INVALID_VALUE;
    if (slope && (Z == nullptr || short_ld(ldz, m))) return RTAT_STATUS_INVALID_VALUE;
    if (slope && q.dZ != nullptr && short_ld(q.lddz, m)) return RTAT_STATUS_INVALID_VALUE;
    if (*alpha != 0.0f) {
      if (slope && q.dZ == nullptr && (want_a || want_b)) return RTAT_STATUS_INVALID_VALUE;
      if (want_a && (B == nullptr || short_ld(ldb, tb ? n : k))) return RTAT_STATUS_INVALID_VALUE;
      if (want_b && (A == nullptr || short_ld(lda, ta ? k : m))) return RTAT_STATUS_INVALID_VALUE;
    }
  }
  OnDevice on(h);
  rtat_status_t st = RTAT_STATUS_SUCCESS;
  if (m > 0 && ((slope && q.dZ != nullptr && n > 0) || q.dbias != nullptr))
    st = launch_act_backward(h, type, act, m, n, dD, lddd, Z, ldz, slope ? q.dZ : nullptr, q.lddz,
                             q.dbias);
  if (st != RTAT_STATUS_SUCCESS) return st;
  const void* dZ = slope ? q.dZ : dD;
  const long lddz = slope ? q.lddz : lddd;
  if (want_a) {
    // op(A) = A: dA (m x k) = dZ op(B)^T;  op(A) = A^T: dA (k x m) = op(B) dZ^T
    Gemm16 g = ta ? product(type, tb, true, k, m, n, *alpha, B, ldb, dZ, lddz)
                  : product(type, false, !tb, m, k, n, *alpha, dZ, lddz, B, ldb);
    g.ep.beta = q.da_beta;
    g.ep.C = q.da_beta != 0.0f ? q.dA : nullptr;
    g.ep.D = q.dA;
    g.ep.ldc = g.ep.ldd = q.ldda;
    g.ep.c_type = g.ep.d_type = q.da_type;
    st = launch_gemm16(h, g);
    if (st != RTAT_STATUS_SUCCESS) return st;
  }
  if (want_b) {
    // op(B) = B: dB (k x n) = op(A)^T dZ;  op(B) = B^T: dB (n x k) = dZ^T op(A)
    Gemm16 g = tb ? product(type, true, ta, n, k, m, *alpha, dZ, lddz, A, lda)
                  : product(type, !ta, false, k, n, m, *alpha, A, lda, dZ, lddz);
    g.ep.beta = q.db_beta;
    g.ep.C = q.db_beta != 0.0f ? q.dB : nullptr;
    g.ep.D = q.dB;
    g.ep.ldc = g.ep.ldd = q.lddb;
    g.ep.c_type = g.ep.d_type = q.db_type;
    st = launch_gemm16(h, g);
  }
  return st;
}

rtat_status_t rtat_gemm_dact(rtat_handle_t h, rtat_type_t type, rtat_operation_t transa,
                             rtat_operation_t transb, int m, int n, int k, const float* alpha,
                             const void* A, int lda, const void* B, int ldb,
                             rtat_activation_t act, const void* Z, int ldz, void* D, int ldd,
                             float* dbias) {
  RTAT_CHECK_HANDLE(h);
  rtat_status_t st = check_product(type, transa, transb, m, n, k, alpha, A, lda, B, ldb);
  if (st != RTAT_STATUS_SUCCESS) return st;
  if (!valid_act(act)) return RTAT_STATUS_INVALID_ENUM;
  if (m == 0) return RTAT_STATUS_SUCCESS;
  OnDevice on(h);
  if (n == 0)  // sums over nothing
    return dbias == nullptr ? RTAT_STATUS_SUCCESS : launch_sum_rows(h, nullptr, 0, m, dbias);
  if (D == nullptr || short_ld(ldd, m)) return RTAT_STATUS_INVALID_VALUE;
  if (act != RTAT_ACT_NONE && (Z == nullptr || short_ld(ldz, m))) return RTAT_STATUS_INVALID_VALUE;
  Gemm16 g = product(type, transa == RTAT_OP_T, transb == RTAT_OP_T, m, n, k, *alpha, A, lda, B, ldb);
  g.ep.slope = 1;
  g.ep.act = act;
  g.ep.aux = act != RTAT_ACT_NONE ? const_cast<void*>(Z) : nullptr;
  g.ep.ldaux = ldz;
  g.ep.D = D;
  g.ep.ldd = ldd;
  g.ep.d_type = type;
  if (dbias == nullptr) return launch_gemm16(h, g);
  g.ep.sums = acquire_sums(h, m, n);
  if (g.ep.sums == nullptr) return RTAT_STATUS_ALLOC_FAILED;
  g.scratch_used = dbias_workspace_bytes(m, n);
  st = launch_gemm16(h, g);
  if (st != RTAT_STATUS_SUCCESS) return st;
  return launch_sum_rows(h, g.ep.sums, h->sum_rows, m, dbias);
}

size_t rtat_dbias_workspace_bytes(int m, int n) { return dbias_workspace_bytes(m, n); }

rtat_status_t rtat_newton_schulz(rtat_handle_t h, rtat_type_t g_type, int m, int n, int batch,
                                 const void* G, int ldg, int64_t stride_g, int steps,
                                 const float* coeffs, float eps, void* O, int ldo,
                                 int64_t stride_o) {
  RTAT_CHECK_HANDLE(h);
  if (!valid_half(g_type) && g_type != RTAT_TYPE_F32) return RTAT_STATUS_INVALID_ENUM;
  if (m < 0 || n < 0 || batch < 0 || steps < 1 || steps > RTAT_NEWTON_SCHULZ_MAX_STEPS ||
      coeffs == nullptr || !(eps >= 0.0f && eps <= 3.402823466e38f))
    return RTAT_STATUS_INVALID_VALUE;
  if (too_long(m, n, 0)) return RTAT_STATUS_NOT_SUPPORTED;
  if (m == 0 || n == 0 || batch == 0) return RTAT_STATUS_SUCCESS;
  if (G == nullptr || O == nullptr || short_ld(ldg, m) || short_ld(ldo, m))
    return RTAT_STATUS_INVALID_VALUE;
  if (batch > 65535) return RTAT_STATUS_INVALID_VALUE;  // a grid dimension
  OnDevice on(h);
  return launch_newton_schulz(h, g_type, m, n, batch, G, ldg, batch > 1 ? stride_g : 0, steps,
                              coeffs, eps, O, ldo, batch > 1 ? stride_o : 0);
}

size_t rtat_newton_schulz_workspace_bytes(int m, int n, int batch) {
  return newton_schulz_workspace_bytes(m, n, batch);
}

const char* rtat_activation_name(int act) {
  switch (act) {
    case RTAT_ACT_NONE: return "none";
    case RTAT_ACT_RELU: return "relu";
    case RTAT_ACT_GELU: return "gelu";
    case RTAT_ACT_GELU_TANH: return "gelu_tanh";
    case RTAT_ACT_SILU: return "silu";
    default: return nullptr;
  }
}

const char* rtat_version(void) { return "rtat-native 0.1 gfx950"; }

}  // extern "C"
