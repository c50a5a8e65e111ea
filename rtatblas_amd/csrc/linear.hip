// The elementwise half of a linear layer's backward pass: dZ = dD * act'(Z) and its row sums
// (the bias gradient) in one pass.
//
// Memory bound: 6 bytes an element (4 without an activation, 2 for the sums alone).  Sixteen
// lanes take 128 neighbouring rows of a column in 16-byte accesses, a workgroup of 256 sixteen
// columns at a time; the columns are cut into chunks so that the grid fills the machine, each
// chunk leaves one row of partial sums and a second small launch adds those in order, so the
// result does not depend on timing.
#include "gemm16.h"

namespace rtat_native {

namespace {

constexpr int ROWS = 128, COLS = 16;  // rows and columns a workgroup holds at a time

struct ActArgs {
  int type, act, m, n, per_chunk;
  const uint16_t* dD;
  long lddd;
  const uint16_t* Z;
  long ldz;
  uint16_t* dZ;
  long lddz;
  float* sums;  // [chunk][m], or null
};

__global__ __launch_bounds__(256) void act_backward_kernel(ActArgs p) {
  __shared__ float part[COLS][ROWS];
  const int t = threadIdx.x, lr = (t % 16) * 8, lc = t / 16;
  const int row = blockIdx.x * ROWS + lr;
  const int first = blockIdx.y * p.per_chunk;
  const int last = p.n - first < p.per_chunk ? p.n : first + p.per_chunk;
  float sums[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[i] = 0.0f;
  const bool slope = p.act != RTAT_ACT_NONE;
  if (row < p.m) {
    if (row + 8 <= p.m) {
#pragma unroll 4
      for (int col = first + lc; col < last; col += COLS) {
        float v[1][8];
        load8(p.type, p.dD, row + (long)col * p.lddd, v[0]);
        if (slope) {
          const u4_t z[1] = {load16(p.Z, 2 * (row + (long)col * p.ldz))};
          act_slopes<1>(p.act, p.type, z, v);
          if (p.dZ != nullptr) store8(p.type, p.dZ, row + (long)col * p.lddz, v[0]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[i] += v[0][i];
      }
    } else {
      for (int col = first + lc; col < last; col += COLS) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (row + i < p.m) {
            float v = load_one(p.type, p.dD, row + i + (long)col * p.lddd);
            if (slope) {
              v *= act_slope(p.act, load_one(p.type, p.Z, row + i + (long)col * p.ldz));
              if (p.dZ != nullptr) store_one(p.type, p.dZ, row + i + (long)col * p.lddz, v);
            }
            sums[i] += v;
          }
      }
    }
  }
  if (p.sums == nullptr) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) part[lc][lr + i] = sums[i];
  __syncthreads();
  if (t < ROWS && blockIdx.x * ROWS + t < (unsigned)p.m) {
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < COLS; ++c) s += part[c][t];
    p.sums[(long)blockIdx.y * p.m + blockIdx.x * ROWS + t] = s;
  }
}

}  // namespace

size_t dbias_workspace_bytes(int m, int n) {
  if (m <= 0 || n <= 0) return 0;
  return (size_t)dact_sum_rows(n) * (size_t)m * sizeof(float) + 256;  // room to align
}

float* acquire_sums(rtat_native_handle* h, int m, int n) {
  const uintptr_t ws = reinterpret_cast<uintptr_t>(acquire_workspace(h, dbias_workspace_bytes(m, n)));
  return reinterpret_cast<float*>((ws + 255) & ~(uintptr_t)255);
}

rtat_status_t launch_act_backward(rtat_native_handle* h, int type, int act, int m, int n,
                                  const void* dD, long lddd, const void* Z, long ldz, void* dZ,
                                  long lddz, float* dbias) {
  ActArgs p = {};
  p.type = type;
  p.act = act;
  p.m = m;
  p.n = n;
  p.dD = static_cast<const uint16_t*>(dD);
  p.lddd = lddd;
  p.Z = static_cast<const uint16_t*>(Z);
  p.ldz = ldz;
  p.dZ = static_cast<uint16_t*>(dZ);
  p.lddz = lddz;
  const long strips = (m + ROWS - 1) / ROWS;
  // Enough chunks for eight workgroups per CU, none shorter than four passes; never more rows of
  // partial sums than dbias_workspace_bytes counts (one per 32 columns).
  const long want = (8L * (h->compute_units > 0 ? h->compute_units : 256) + strips - 1) / strips;
  long chunks = (n + 4 * COLS - 1) / (4 * COLS);
  if (chunks > want) chunks = want;
  if (chunks < 1) chunks = 1;
  p.per_chunk = (int)((n + chunks - 1) / chunks);
  chunks = n > 0 ? (n + p.per_chunk - 1) / p.per_chunk : 1;
  if (dbias != nullptr) {
    p.sums = dbias;
    if (chunks > 1) {
      p.sums = acquire_sums(h, m, n);
      if (p.sums == nullptr) return RTAT_STATUS_ALLOC_FAILED;
    }
  }
  hipLaunchKernelGGL(act_backward_kernel, dim3((unsigned)strips, (unsigned)chunks), dim3(256), 0,
                     h->stream, p);
  rtat_status_t st = launch_status();
  if (st != RTAT_STATUS_SUCCESS || dbias == nullptr || chunks == 1) return st;
  return launch_sum_rows(h, p.sums, (int)chunks, m, dbias);
}

}  // namespace rtat_native
