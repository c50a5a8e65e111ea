// Newton-Schulz orthogonalisation (rtat_newton_schulz): X <- a X + (b M + c M^2) X, M = X X^T,
// as three products a step on the 16-bit core (gemm16.hip).
//
// What it needs per step, with lo <= hi the two sides: lo^2 hi flop for M (symmetric: half of
// the product), lo^3 for M^2 (symmetric again, with b M + c M^2 formed in its epilogue) and
// 2 lo^2 hi for the product with X, whose epilogue adds a X.  Matrix-core bound for large sides,
// launch bound for small ones.
//
// Precision.  X and M are f16 (11 bits) rather than bf16 (8): both run at the same rate, and all
// values are bounded, so a fixed scale keeps them in range: X by 2^10 (|x| <= singular value, so
// up to 60 fits; entries of size 2^-24 relative to the norm are still normal numbers), M by 2^10,
// b M + c M^2 by 2^8.  A rounding of X in an early step is amplified by a^(steps left) in weak
// directions, so early steps add a X from an f32 copy (step 0 from G itself); only in the last
// two, where singular values have grown to the order of one, is X taken as rounded.  Relative
// error of the result in 2-norm against 64 bits, sides 128 .. 1024, five steps, four spectra
// (Gaussian, rank 16 over a floor of 10 % and of 1 %, power law): at most 1.5e-3 that way,
// 1.7e-2 without the f32 copies, 0.13 with bf16; rounding the result to bf16 is 1.7e-3.
// The norm is summed in f64.  G is scaled by a power of two when it becomes f16, so a 16-bit G
// does not round; what is left of the norm (r in [1, 2)) enters the scalars of step 0.
//
// Sides are padded with zeros to multiples of 64 in the scratch, which leaves the products
// unchanged and every operand aligned.
#include "gemm16.h"

namespace rtat_native {

namespace {

constexpr float X_SCALE = 1024.0f, M_SCALE = 1024.0f, P_SCALE = 256.0f;
constexpr int NORM_BLOCKS = 1024;  // partial sums per matrix, at most

struct NormArgs {
  int type, m, n, mp, np, blocks;
  const void* G;
  long ldg, stride_g;
  float eps;
  double* parts;  // [matrix][blocks]
  float* scale;   // [matrix]{r, e}
  uint16_t* X;    // f16, mp x np
  long x_stride;
};

__device__ inline double block_sum(double s, double* lds) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2) s += __shfl_xor(s, d);
  const int wave = threadIdx.x / 64;
  if (threadIdx.x % 64 == 0) lds[wave] = s;
  __syncthreads();
  return lds[0] + lds[1] + lds[2] + lds[3];
}

// Eight rows of a column from `row` on; rows past m read as zero.
__device__ inline void rows8(const NormArgs& p, long at, int row, float (&v)[8]) {
  if (row + 8 <= p.m) {
    load8(p.type, p.G, at + row, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = row + i < p.m ? load_one(p.type, p.G, at + row + i) : 0.0f;
  }
}

// Partial sums of squares: a matrix is cut into pieces of eight rows of a column, dealt to the
// threads of all blocks in turn.
__global__ __launch_bounds__(256) void norm_kernel(NormArgs p) {
  __shared__ double lds[4];
  const long z = blockIdx.y, per_col = (p.m + 7) / 8, pieces = per_col * p.n;
  const long step = 256L * p.blocks;
  double s = 0.0;
#pragma unroll 4
  for (long i = blockIdx.x * 256L + threadIdx.x; i < pieces; i += step) {
    const long col = i / per_col;
    float v[8];
    rows8(p, z * p.stride_g + col * p.ldg, (int)(i - col * per_col) * 8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += (double)v[e] * (double)v[e];
  }
  s = block_sum(s, lds);
  if (threadIdx.x == 0) p.parts[z * p.blocks + blockIdx.x] = s;
}

// X = f16(2^e G), 2^e the power of two at or below X_SCALE / norm, zeros in the padding.
__global__ __launch_bounds__(256) void scale_kernel(NormArgs p) {
  __shared__ double lds[4];
  const long z = blockIdx.y;
  double s = 0.0;
  for (int i = threadIdx.x; i < p.blocks; i += 256) s += p.parts[z * p.blocks + i];
  s = block_sum(s, lds);
  const double want = (double)X_SCALE / (sqrt(s) + (double)p.eps);
  // want is 0 or NaN for a G that holds an infinity or a NaN, infinite for a zero norm: the
  // ratio r then is NaN, and through it every element of the result.
  int e = 0;
  double r = want - want;  // NaN unless finite
  if (want > 0.0 && r == 0.0) {
    e = ilogb(want);
    r = ldexp(want, -e);
  } else {
    r = __builtin_nan("");
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.scale[2 * z] = (float)r;
    p.scale[2 * z + 1] = (float)e;
  }
  uint16_t* X = p.X + z * p.x_stride;
  const long per_col = p.mp / 8, pieces = per_col * p.np, step = 256L * gridDim.x;
#pragma unroll 4
  for (long i = blockIdx.x * 256L + threadIdx.x; i < pieces; i += step) {
    const long col = i / per_col;
    const int row = (int)(i - col * per_col) * 8;
    float v[8];
    if (col < p.n && row < p.m) {
      rows8(p, z * p.stride_g + col * p.ldg, row, v);
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = 0.0f;
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = __builtin_ldexpf(v[q], e);
    store8(RTAT_TYPE_F16, X, row + col * p.mp, v);
  }
}

struct Layout {
  long mp, np, lp;  // padded sides, the shorter of them
  size_t x, p, parts, scale, total;  // bytes per matrix of X and M; offsets
};

inline size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

Layout layout_of(int m, int n, int batch) {
  Layout l;
  l.mp = ((long)m + 63) / 64 * 64;
  l.np = ((long)n + 63) / 64 * 64;
  l.lp = m <= n ? l.mp : l.np;
  l.x = (size_t)l.mp * (size_t)l.np;  // elements
  l.p = (size_t)l.lp * (size_t)l.lp;
  size_t at = 0;
  at += align256((size_t)batch * l.x * 2) * 2;  // two f16 X
  at += align256((size_t)batch * l.x * 4);      // the f32 copy
  at += align256((size_t)batch * l.p * 2) * 2;  // M and its polynomial
  l.parts = at;
  at += align256((size_t)batch * NORM_BLOCKS * sizeof(double));
  l.scale = at;
  at += align256((size_t)batch * 2 * sizeof(float));
  l.total = at;
  return l;
}

}  // namespace

size_t newton_schulz_workspace_bytes(int m, int n, int batch) {
  if (m <= 0 || n <= 0 || batch <= 0) return 0;
  return layout_of(m, n, batch).total + 256;
}

rtat_status_t launch_newton_schulz(rtat_native_handle* h, int g_type, int m, int n, int batch,
                                   const void* G, long ldg, long stride_g, int steps,
                                   const float* coeffs, float eps, void* O, long ldo,
                                   long stride_o) {
  const Layout l = layout_of(m, n, batch);
  unsigned char* ws =
      static_cast<unsigned char*>(acquire_workspace(h, newton_schulz_workspace_bytes(m, n, batch)));
  if (ws == nullptr) return RTAT_STATUS_ALLOC_FAILED;
  ws = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(ws) + 255) & ~(uintptr_t)255);
  const size_t xb = align256((size_t)batch * l.x * 2), pb = align256((size_t)batch * l.p * 2);
  uint16_t* X[2] = {reinterpret_cast<uint16_t*>(ws), reinterpret_cast<uint16_t*>(ws + xb)};
  float* F = reinterpret_cast<float*>(ws + 2 * xb);
  unsigned char* after = ws + 2 * xb + align256((size_t)batch * l.x * 4);
  uint16_t* M = reinterpret_cast<uint16_t*>(after);
  uint16_t* P = reinterpret_cast<uint16_t*>(after + pb);
  float* scale = reinterpret_cast<float*>(ws + l.scale);

  NormArgs a = {};
  a.type = g_type;
  a.m = m;
  a.n = n;
  a.mp = (int)l.mp;
  a.np = (int)l.np;
  auto blocks_for = [](long pieces) {  // two pieces a thread
    const long b = (pieces + 511) / 512;
    return (int)(b < NORM_BLOCKS ? b : NORM_BLOCKS);
  };
  a.blocks = blocks_for((((long)m + 7) / 8) * n);
  a.G = G;
  a.ldg = ldg;
  a.stride_g = stride_g;
  a.eps = eps;
  a.parts = reinterpret_cast<double*>(ws + l.parts);
  a.scale = scale;
  a.X = X[0];
  a.x_stride = (long)l.x;
  hipLaunchKernelGGL(norm_kernel, dim3((unsigned)a.blocks, (unsigned)batch), dim3(256), 0,
                     h->stream, a);
  rtat_status_t st = launch_status();
  if (st != RTAT_STATUS_SUCCESS) return st;
  hipLaunchKernelGGL(scale_kernel, dim3((unsigned)blocks_for(l.mp / 8 * l.np), (unsigned)batch), dim3(256), 0, h->stream, a);
  st = launch_status();
  if (st != RTAT_STATUS_SUCCESS) return st;

  const bool wide = m <= n;  // M = X X^T, else X^T X
  for (int i = 0; i < steps; ++i) {
    const float ca = coeffs[3 * i], cb = coeffs[3 * i + 1], cc = coeffs[3 * i + 2];
    const bool last = i == steps - 1;
    // M
    Gemm16 g = {};
    g.type = RTAT_TYPE_F16;
    g.batch = batch;
    g.tri = 1;
    g.ta = !wide;
    g.tb = wide;
    g.m = g.n = (int)l.lp;
    g.k = (int)(wide ? l.np : l.mp);
    g.A = g.B = X[i & 1];
    g.lda = g.ldb = l.mp;
    g.a_stride = g.b_stride = (long)l.x;
    Epilogue e = {};
    e.rows = e.cols = (int)l.lp;
    e.alpha = M_SCALE / (X_SCALE * X_SCALE);
    e.D = M;
    e.ldd = l.lp;
    e.d_stride = (long)l.p;
    e.d_type = RTAT_TYPE_F16;
    if (i == 0) {
      e.scale = scale;
      e.r_power = 2;
    }
    g.ep = e;
    st = launch_gemm16(h, g);
    if (st != RTAT_STATUS_SUCCESS) return st;
    // P = b M + c M^2
    g.ta = true;
    g.tb = false;
    g.k = (int)l.lp;
    g.A = g.B = M;
    g.lda = g.ldb = l.lp;
    g.a_stride = g.b_stride = (long)l.p;
    e.scale = nullptr;
    e.r_power = 0;
    e.alpha = cc * P_SCALE / (M_SCALE * M_SCALE);
    e.beta = cb * P_SCALE / M_SCALE;
    e.C = M;
    e.ldc = l.lp;
    e.c_stride = (long)l.p;
    e.c_type = RTAT_TYPE_F16;
    e.c_rows = e.c_cols = (int)l.lp;
    e.D = P;
    g.ep = e;
    st = launch_gemm16(h, g);
    if (st != RTAT_STATUS_SUCCESS) return st;
    // X = a X + P X (X P when M = X^T X)
    g.tri = 0;
    g.ta = wide;
    g.tb = false;
    g.A = wide ? P : X[i & 1];
    g.B = wide ? X[i & 1] : P;
    g.lda = wide ? l.lp : l.mp;
    g.ldb = wide ? l.mp : l.lp;
    g.a_stride = (long)(wide ? l.p : l.x);
    g.b_stride = (long)(wide ? l.x : l.p);
    g.m = (int)l.mp;
    g.n = (int)l.np;
    g.k = (int)l.lp;
    e = Epilogue{};
    const float out = last ? 1.0f / X_SCALE : 1.0f;
    e.alpha = out / P_SCALE;
    e.beta = ca * out;
    if (i == 0) {  // C = G, as r 2^e G
      e.scale = scale;
      e.r_power = 1;
      e.scale_c = 1;
      e.C = G;
      e.ldc = ldg;
      e.c_stride = stride_g;
      e.c_type = g_type;
      e.c_rows = m;
      e.c_cols = n;
    } else {
      const bool f32 = i < steps - 2;
      e.C = f32 ? static_cast<const void*>(F) : X[i & 1];
      e.c_type = f32 ? RTAT_TYPE_F32 : RTAT_TYPE_F16;
      e.ldc = l.mp;
      e.c_stride = (long)l.x;
      e.c_rows = (int)l.mp;
      e.c_cols = (int)l.np;
    }
    if (last) {
      g.m = e.rows = m;
      g.n = e.cols = n;
      e.D = O;
      e.ldd = ldo;
      e.d_stride = stride_o;
      e.d_type = RTAT_TYPE_BF16;
    } else {
      e.rows = (int)l.mp;
      e.cols = (int)l.np;
      e.ldd = l.mp;
      e.d_stride = (long)l.x;
      if (i + 1 < steps - 2) {
        e.D = F;
        e.d_type = RTAT_TYPE_F32;
        e.copy = X[(i + 1) & 1];
        e.ldcopy = l.mp;
        e.copy_stride = (long)l.x;
      } else {
        e.D = X[(i + 1) & 1];
        e.d_type = RTAT_TYPE_F16;
      }
    }
    g.ep = e;
    st = launch_gemm16(h, g);
    if (st != RTAT_STATUS_SUCCESS) return st;
  }
  return RTAT_STATUS_SUCCESS;
}

}  // namespace rtat_native
