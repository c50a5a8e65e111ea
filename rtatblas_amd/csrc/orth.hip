// Newton-Schulz orthogonalisation (rtat_newton_schulz): X <- a X + (b M + c M^2) X, M = X X^T,
// as three products a step on the 16-bit core (gemm16.hip).
//
// What it needs per step, with lo <= hi the two sides: lo^2 hi flop for M (symmetric: half of
// the product), lo^3 for M^2 (symmetric again, with b M + c M^2 formed in its epilogue) and
// 2 lo^2 hi for the product with X, whose epilogue adds a X.  Matrix-core bound for large sides,
// launch bound for small ones.
//
// Layout.  X is kept hi x lo, contiguous along its long side, whichever way round G is: M = X^T X
// then has both operands contiguous along k, and X M only one that is not (two in M, none in
// M X, the other way round; an operand that is not costs two transposing LDS reads for one).  A
// G with m < n is transposed when it is scaled, and the last step, which writes O, computes the
// transpose of its product.  Sides are padded with zeros to multiples of 64, which leaves the
// products unchanged and every operand aligned.
//
// Precision.  X and M are f16 (11 bits) rather than bf16 (8): both run at the same rate, and all
// values are bounded, so a fixed scale keeps them in range: X by 2^10 (|x| <= singular value, so
// up to 60 fits; entries of size 2^-24 relative to the norm are still normal numbers), M by 2^10,
// b M + c M^2 by 2^8.  A rounding of X in an early step is amplified by a^(steps left) in weak
// directions, so early steps add a X from an f32 copy (or from a 16-bit G, which f16 holds
// exactly); in the last two, where singular values have grown to the order of one, a joins the
// diagonal of the polynomial instead.  Relative error of the result in 2-norm against 64 bits,
// sides 128 .. 1024, five steps, four spectra (Gaussian, rank 16 over a floor of 10 % and of 1 %,
// power law), emulated: at most 1.5e-3 that way, 1.7e-2 without the f32 copies, 0.13 with bf16;
// rounding the result to bf16 is 1.7e-3.
// The norm is summed in f64.  G is scaled by a power of two when it becomes f16, so a 16-bit G
// does not round; what is left of the norm (r in [1, 2)) enters the scalars of step 0.
#include "gemm16.h"

namespace rtat_native {

namespace {

constexpr float X_SCALE = 1024.0f, M_SCALE = 1024.0f, P_SCALE = 256.0f;
constexpr int NORM_BLOCKS = 1024;  // partial sums per matrix, at most

struct NormArgs {
  int type, m, n, blocks;
  const void* G;
  long ldg, stride_g;
  float eps;
  double* parts;  // [matrix][blocks]
  float* scale;   // [matrix]: r
  int xr, xc;     // padded rows and columns of X
  uint16_t* X;    // f16
  float* F;       // the same in f32, or null
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

// The power of two 2^e at or below X_SCALE / norm, and the ratio r that is left.  The ratio is NaN,
// and through it every element of the result, for a G that holds an infinity or a NaN (the quotient
// is 0 or NaN) and for a zero norm without eps (infinite).
__device__ inline int norm_exponent(const NormArgs& p, long z, double* lds, double& r) {
  double s = 0.0;
  for (int i = threadIdx.x; i < p.blocks; i += 256) s += p.parts[z * p.blocks + i];
  s = block_sum(s, lds);
  const double want = (double)X_SCALE / (sqrt(s) + (double)p.eps);
  if (!(want > 0.0) || want - want != 0.0) {
    r = __builtin_nan("");
    return 0;
  }
  const int e = ilogb(want);
  r = ldexp(want, -e);
  return e;
}

__device__ inline void put_x(const NormArgs& p, long z, int row, int col, int e, float (&v)[8]) {
#pragma unroll
  for (int q = 0; q < 8; ++q) v[q] = __builtin_ldexpf(v[q], e);
  const long at = z * p.x_stride + row + (long)col * p.xr;
  store8(RTAT_TYPE_F16, p.X, at, v);
  if (p.F != nullptr) store8(RTAT_TYPE_F32, p.F, at, v);
}

// X = f16(2^e G), zeros in the padding.
__global__ __launch_bounds__(256) void scale_kernel(NormArgs p) {
  __shared__ double lds[4];
  const long z = blockIdx.y;
  double r;
  const int e = norm_exponent(p, z, lds, r);
  if (blockIdx.x == 0 && threadIdx.x == 0) p.scale[z] = (float)r;
  const int per_col = p.xr / 8;
  const long pieces = (long)per_col * p.xc, step = 256L * gridDim.x;
#pragma unroll 4
  for (long i = blockIdx.x * 256L + threadIdx.x; i < pieces; i += step) {
    const int col = (int)(i / per_col), row = (int)(i - (long)col * per_col) * 8;
    float v[8];
    if (col < p.n && row < p.m) {
      rows8(p, z * p.stride_g + (long)col * p.ldg, row, v);
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = 0.0f;
    }
    put_x(p, z, row, col, e, v);
  }
}

// X = f16(2^e G^T): a workgroup turns 64 x 64 blocks over through LDS.
__global__ __launch_bounds__(256) void turn_kernel(NormArgs p) {
  __shared__ double lds[4];
  __shared__ float block[64][65];
  const long z = blockIdx.y;
  double r;
  const int e = norm_exponent(p, z, lds, r);
  if (blockIdx.x == 0 && threadIdx.x == 0) p.scale[z] = (float)r;
  const int t = threadIdx.x, across = p.xc / 64;
  const long blocks = (long)(p.xr / 64) * across;
  for (long b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int x_row = (int)(b / across) * 64, x_col = (int)(b % across) * 64;
    // Rows x_col .. + 63 of G's columns x_row .. + 63, eight at a time.
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int g = (t & 7) * 8, c = (t >> 3) + 32 * h;
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = 0.0f;
      if (x_row + c < p.n && x_col + g < p.m)
        rows8(p, z * p.stride_g + (long)(x_row + c) * p.ldg, x_col + g, v);
#pragma unroll
      for (int q = 0; q < 8; ++q) block[g + q][c] = v[q];
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = (t & 7) * 8, col = (t >> 3) + 32 * h;
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = block[col][row + q];
      put_x(p, z, x_row + row, x_col + col, e, v);
    }
    __syncthreads();
  }
}

struct Layout {
  long hp, lp;                                 // padded sides, the longer first
  size_t x, p;                                 // elements of X and of M
  size_t x1, f, mm, pp, parts, scale, total;   // byte offsets behind the first X
};

inline size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

Layout layout_of(int m, int n, int batch) {
  Layout l;
  const long mp = ((long)m + 63) / 64 * 64, np = ((long)n + 63) / 64 * 64;
  l.hp = mp > np ? mp : np;
  l.lp = mp > np ? np : mp;
  l.x = (size_t)l.hp * (size_t)l.lp;
  l.p = (size_t)l.lp * (size_t)l.lp;
  const size_t b = (size_t)batch;
  l.x1 = align256(b * l.x * 2);
  l.f = 2 * l.x1;
  l.mm = l.f + align256(b * l.x * 4);
  l.pp = l.mm + align256(b * l.p * 2);
  l.parts = l.pp + align256(b * l.p * 2);
  l.scale = l.parts + align256(b * NORM_BLOCKS * sizeof(double));
  l.total = l.scale + align256(b * sizeof(float));
  return l;
}

// One product of a step on matrices of the scratch.
Gemm16 step_product(int batch, int m, int n, int k, bool ta, bool tb, const void* A, long lda,
                    long a_stride, const void* B, long ldb, long b_stride, float alpha, void* D,
                    long ldd, long d_stride, int d_type) {
  Gemm16 g = {};
  g.type = RTAT_TYPE_F16;
  g.batch = batch;
  g.m = g.ep.rows = m;
  g.n = g.ep.cols = n;
  g.k = k;
  g.ta = ta;
  g.tb = tb;
  g.A = A;
  g.lda = lda;
  g.a_stride = a_stride;
  g.B = B;
  g.ldb = ldb;
  g.b_stride = b_stride;
  g.ep.alpha = alpha;
  g.ep.D = D;
  g.ep.ldd = ldd;
  g.ep.d_stride = d_stride;
  g.ep.d_type = d_type;
  return g;
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
  uint16_t* const X[2] = {reinterpret_cast<uint16_t*>(ws), reinterpret_cast<uint16_t*>(ws + l.x1)};
  float* const F = reinterpret_cast<float*>(ws + l.f);
  uint16_t* const M = reinterpret_cast<uint16_t*>(ws + l.mm);
  uint16_t* const P = reinterpret_cast<uint16_t*>(ws + l.pp);
  float* const scale = reinterpret_cast<float*>(ws + l.scale);
  const int hp = (int)l.hp, lp = (int)l.lp;
  const long xs = (long)l.x, ps = (long)l.p;
  const bool turn = (m + 63) / 64 < (n + 63) / 64;  // X is G^T
  // Whether step i adds a X rather than putting a on the polynomial's diagonal.
  auto adds = [&](int i) { return i < steps - 2; };

  NormArgs a = {};
  a.type = g_type;
  a.m = m;
  a.n = n;
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
  a.xr = hp;
  a.xc = lp;
  a.X = X[0];
  a.F = g_type == RTAT_TYPE_F32 && adds(0) ? F : nullptr;
  a.x_stride = xs;
  hipLaunchKernelGGL(norm_kernel, dim3((unsigned)a.blocks, (unsigned)batch), dim3(256), 0,
                     h->stream, a);
  rtat_status_t st = launch_status();
  if (st != RTAT_STATUS_SUCCESS) return st;
  if (turn) {
    const long blocks = l.hp / 64 * (l.lp / 64);
    hipLaunchKernelGGL(turn_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048), (unsigned)batch),
                       dim3(256), 0, h->stream, a);
  } else {
    hipLaunchKernelGGL(scale_kernel, dim3((unsigned)blocks_for((long)l.x / 8), (unsigned)batch),
                       dim3(256), 0, h->stream, a);
  }
  st = launch_status();
  if (st != RTAT_STATUS_SUCCESS) return st;

  for (int i = 0; i < steps; ++i) {
    const float ca = coeffs[3 * i], cb = coeffs[3 * i + 1], cc = coeffs[3 * i + 2];
    const bool last = i == steps - 1;
    const uint16_t* const x = X[i & 1];
    uint16_t* const y = X[(i + 1) & 1];
    // M = X^T X
    Gemm16 g = step_product(batch, lp, lp, hp, true, false, x, hp, xs, x, hp, xs,
                            M_SCALE / (X_SCALE * X_SCALE), M, lp, ps, RTAT_TYPE_F16);
    g.tri = 1;
    if (i == 0) {
      g.ep.scale = scale;
      g.ep.r_power = 2;
    }
    st = launch_gemm16(h, g);
    if (st != RTAT_STATUS_SUCCESS) return st;
    // P = b M + c M^2 (+ a)
    g = step_product(batch, lp, lp, lp, true, false, M, lp, ps, M, lp, ps,
                     cc * P_SCALE / (M_SCALE * M_SCALE), P, lp, ps, RTAT_TYPE_F16);
    g.tri = 1;
    g.ep.beta = cb * P_SCALE / M_SCALE;
    g.ep.C = M;
    g.ep.ldc = lp;
    g.ep.c_stride = ps;
    g.ep.c_type = RTAT_TYPE_F16;
    g.ep.diag = adds(i) ? 0.0f : ca * P_SCALE;
    st = launch_gemm16(h, g);
    if (st != RTAT_STATUS_SUCCESS) return st;
    // X = X P (+ a X)
    if (!last) {
      g = step_product(batch, hp, lp, lp, false, false, x, hp, xs, P, lp, ps, 1.0f / P_SCALE, y, hp,
                       xs, RTAT_TYPE_F16);
      if (adds(i)) {
        const bool f32 = i > 0 || a.F != nullptr;
        g.ep.beta = ca;
        g.ep.C = f32 ? static_cast<const void*>(F) : x;
        g.ep.ldc = hp;
        g.ep.c_stride = xs;
        g.ep.c_type = f32 ? RTAT_TYPE_F32 : RTAT_TYPE_F16;
      }
      if (adds(i + 1)) {  // an f32 copy for the next step, over the one just read
        g.ep.copy = y;
        g.ep.ldcopy = hp;
        g.ep.copy_stride = xs;
        g.ep.D = F;
        g.ep.d_type = RTAT_TYPE_F32;
      }
    } else if (turn) {  // O = (X P)^T = P X^T
      g = step_product(batch, m, n, lp, true, true, P, lp, ps, x, hp, xs, 1.0f / (P_SCALE * X_SCALE),
                       O, ldo, stride_o, RTAT_TYPE_BF16);
    } else {
      g = step_product(batch, m, n, lp, false, false, x, hp, xs, P, lp, ps,
                       1.0f / (P_SCALE * X_SCALE), O, ldo, stride_o, RTAT_TYPE_BF16);
    }
    if (i == 0) {
      g.ep.scale = scale;
      g.ep.r_power = 1;
      g.ep.scale_c = 1;
    }
    st = launch_gemm16(h, g);
    if (st != RTAT_STATUS_SUCCESS) return st;
  }
  return RTAT_STATUS_SUCCESS;
}

}  // namespace rtat_native
