// The elementwise half of a linear layer's backward pass: dZ = dD * act'(Z) and its row sums
// (the bias gradient) in one pass.
//
// Memory bound: 6 bytes an element (4 without an activation, 2 for the sums alone).  Sixteen
// lanes take 128 neighbouring rows of a column in 16-byte accesses, a workgroup of 256 sixteen
// columns at a time; the columns are cut into chunks so that the grid fills the machine, each
// chunk leaves one row of partial sums and a second small launch adds those in order, so the
// result does not depend on timing.  Four groups of columns on their way before the first store:
// 6580 x 4711 f16 on 8-byte aligned columns 62 -> 47 us, 413 x 456 20 -> 12.
#include <type_traits>

#include "gemm16.h"

namespace rtat_native {

namespace {

constexpr int ROWS = 128, COLS = 16;  // rows and columns a workgroup holds at a time
constexpr int AHEAD = 4;              // that many times COLS are on their way

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

// Eight neighbours, of which the first `left` >= 1 are there; the others read as zero.  Without
// branches, so that loads of several columns overlap.
template <bool PART>
__device__ inline u4_t fetch8(const uint16_t* p, long i, int left) {
  if (!PART) return load16(p, 2 * i);
  s8_t v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (short)p[i + (e < left ? e : left - 1)];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e < left ? v[e] : (short)0;
  return __builtin_bit_cast(u4_t, v);
}

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
  const int left = p.m - row;
  auto columns = [&](auto part) {
    constexpr bool PART = decltype(part)::value;
    // Four columns are asked for before the first is stored: dZ may be dD, so the compiler would
    // not move a load over a store by itself.
    for (int col = first + lc; col < last; col += AHEAD * COLS) {
      u4_t d[AHEAD], z[AHEAD][1];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int c = col + u * COLS < last ? col + u * COLS : last - 1;  // its sums are left out
        d[u] = fetch8<PART>(p.dD, row + (long)c * p.lddd, left);
        z[u][0] = slope ? fetch8<PART>(p.Z, row + (long)c * p.ldz, left) : u4_t{};
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int c = col + u * COLS;
        if (c >= last) break;
        float v[1][8];
        unpack8(p.type, d[u], v[0]);
        if (slope) {
          act_slopes<1>(p.act, p.type, z[u], v);
          if (p.dZ != nullptr) {
            if (PART) store8_part(p.type, p.dZ, row + (long)c * p.lddz, left, v[0]);
            else store8(p.type, p.dZ, row + (long)c * p.lddz, v[0]);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[i] += v[0][i];
      }
    }
  };
  if (left >= 8) columns(std::false_type());
  else if (left > 0) columns(std::true_type());
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
