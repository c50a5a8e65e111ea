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
// values are bounded, so scales keep them in range: X by 2^10 (|x| <= singular value, so up to 60
// fits; the norm of the first X lies in (512, 1024], so entries down to 2^-24 of it are within a
// factor of two of f16's smallest normal number), M by at most 2^10 and b M + c M^2 by at most 2^8, as far
// as a bound on the singular values leaves room (orth_plan.h).
// A rounding of X in an early step is amplified by a^(steps left) in weak
// directions, so early steps add a X from an f32 copy (or from a 16-bit G, which f16 holds
// exactly); in the last two, where singular values have grown to the order of one, a joins the
// diagonal of the polynomial instead.  Relative error of the result in 2-norm against 64 bits,
// sides 128 .. 1024, five steps, four spectra (Gaussian, rank 16 over a floor of 10 % and of 1 %,
// power law), emulated: at most 1.5e-3 that way, 1.7e-2 without the f32 copies, 0.13 with bf16;
// rounding the result to bf16 is 1.7e-3.
// The norm is summed in f64.  G is scaled by a power of two when it becomes f16, so a 16-bit G
// does not round; what is left of the norm (r in [1, 2)) enters the scalars of step 0.
#include "gemm16.h"
#include "orth_plan.h"

namespace rtat_native {

namespace {

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

// Sum over a workgroup of WAVES waves, the same order in every thread.
template <int WAVES>
__device__ inline double block_sum(double s, double* lds) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2) s += __shfl_xor(s, d);
  const int wave = threadIdx.x / 64;
  if (threadIdx.x % 64 == 0) lds[wave] = s;
  __syncthreads();
  s = lds[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) s += lds[w];
  return s;
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
  s = block_sum<4>(s, lds);
  if (threadIdx.x == 0) p.parts[z * p.blocks + blockIdx.x] = s;
}

// The power of two 2^e at or below `want` = X_SCALE / norm, and the ratio r that is left.  The ratio
// is NaN, and through it every element of the result, for a G that holds an infinity or a NaN (the
// quotient is 0 or NaN) and for a zero norm without eps (infinite).
__device__ inline int exponent_of(double want, double& r) {
  if (!(want > 0.0) || want - want != 0.0) {
    r = __builtin_nan("");
    return 0;
  }
  const int e = ilogb(want);
  r = ldexp(want, -e);
  return e;
}
__device__ inline int norm_exponent(const NormArgs& p, long z, double* lds, double& r) {
  double s = 0.0;
  for (int i = threadIdx.x; i < p.blocks; i += 256) s += p.parts[z * p.blocks + i];
  s = block_sum<4>(s, lds);
  return exponent_of((double)X_SCALE / (sqrt(s) + (double)p.eps), r);
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

// ---- sides of at most 128: the whole iteration in one workgroup --------------------------------
//
// At these sizes the products take less time than the launches between them (128 x 128, five
// steps: 17 launches 95 us), so a workgroup keeps a matrix to itself: X, M and P in LDS as SIDE
// rows of SIDE f16, X besides in registers in f32, where the waves' accumulators lie anyway (eight
// wave tiles of SIDE / 2 by SIDE / 4, the same place in every product).  M and P are whole: the
// half that symmetry would save is not worth the extra steps.  128 x 128, five steps: 29 us with
// eight waves, 34 with four, which have half as many requests for LDS on their way.
//
// LDS rows are the short side of X, so X^T X reads both operands as they lie and X P reads X
// transposing.  Chunk c of row r lies at c ^ key(r): eight rows that are read together, or the
// eight rows of a transposing read, fall on different banks.
constexpr int SMALL_THREADS = 512;
struct SmallArgs {
  NormArgs g;  // G; no scratch
  int turn;    // 1: X is G^T
  int steps;
  uint16_t* O;
  long ldo, stride_o;
  StepFactors step[RTAT_NEWTON_SCHULZ_MAX_STEPS];
};

template <int SIDE>
struct Square {
  static constexpr int ROW = SIDE * 2, BYTES = SIDE * ROW;
  static constexpr int TM = SIDE / 32, TN = SIDE / 64;  // blocks of a wave tile
  __device__ static inline int key(int r) {
    if (SIDE == 128) return 2 * ((r & 3) | ((r >> 1) & 4)) | ((r >> 2) & 1);
    return 2 * (((r >> 1) & 1) | ((r >> 2) & 2)) | ((r >> 2) & 1);
  }
  // Byte of element k (a multiple of 4) of row r.
  __device__ static inline int at(int r, int k) {
    return r * ROW + (((k >> 3) ^ key(r)) * 16) + (k & 4) * 2;
  }
  // MFMA operand: sixteen rows from `row` on, K-step `step`.
  __device__ static inline s8_t rows(const unsigned char* x, int row, int step, int lane) {
    return *reinterpret_cast<const s8_t*>(x + at(row + (lane & 15), 32 * step + 8 * (lane >> 4)));
  }
  // ... sixteen columns from `col` on: k runs down the rows.
  __device__ static inline s8_t cols(const unsigned char* x, int col, int step, int lane) {
    typedef __attribute__((address_space(3))) s4_t* lds4_t;
    const int k = 32 * step + 8 * (lane >> 4) + ((lane & 15) >> 2), c = col + 4 * (lane & 3);
    const s4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(x + at(k, c)));
    const s4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(x + at(k + 4, c)));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // acc = (rows or columns of A) times (rows of B) for the wave tile at (m0, n0).
  template <bool COLS>
  __device__ static inline void multiply(const unsigned char* A, const unsigned char* B, int m0,
                                         int n0, int lane, f4_t (&acc)[TM][TN]) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f4_t{0, 0, 0, 0};
#pragma unroll
    for (int step = 0; step < SIDE / 32; ++step) {
      s8_t a[TM], b[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i)
        a[i] = COLS ? cols(A, m0 + 16 * i, step, lane) : rows(A, m0 + 16 * i, step, lane);
#pragma unroll
      for (int j = 0; j < TN; ++j) b[j] = rows(B, n0 + 16 * j, step, lane);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = Half<_Float16>::mfma(a[i], b[j], acc[i][j]);
    }
  }
  // Four neighbouring elements of row r in f16.
  __device__ static inline void put(unsigned char* x, int r, int k, const f4_t& v) {
    typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
    *reinterpret_cast<h4_t*>(x + at(r, k)) =
        h4_t{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
  }
  __device__ static inline f4_t get(const unsigned char* x, int r, int k) {
    typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
    const h4_t h = *reinterpret_cast<const h4_t*>(x + at(r, k));
    return f4_t{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
  }
};

template <int SIDE>
__global__ __launch_bounds__(SMALL_THREADS) void small_kernel(SmallArgs p) {
  typedef Square<SIDE> Q;
  constexpr int TM = Q::TM, TN = Q::TN, NT = SMALL_THREADS;
  extern __shared__ __align__(16) unsigned char lds[];
  __shared__ double sums[NT / 64];
  unsigned char *X = lds, *M = lds + Q::BYTES, *P = lds + 2 * Q::BYTES;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int m0 = (wave & 1) * (SIDE / 2), n0 = (wave >> 1) * (SIDE / 4);
  const long z = blockIdx.x, g0 = z * p.g.stride_g;
  // This lane's accumulators: rows (of the long side) hi0 + 16 i .. + 3, columns lo0 + 16 j.
  const int hi0 = m0 + 4 * (lane >> 4), lo0 = n0 + (lane & 15);

  // G in pieces of eight rows of a column: their squares, then X.
  constexpr int PIECES = SIDE * SIDE / 8 / NT;
  float v[PIECES][8];
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int piece = i * NT + t, row = piece % (SIDE / 8) * 8, col = piece / (SIDE / 8);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[i][q] = 0.0f;
    if (col < p.g.n && row < p.g.m) rows8(p.g, g0 + (long)col * p.g.ldg, row, v[i]);
  }
#pragma unroll
  for (int i = 0; i < PIECES; ++i)
#pragma unroll
    for (int q = 0; q < 8; ++q) s += (double)v[i][q] * (double)v[i][q];
  s = block_sum<NT / 64>(s, sums);
  double ratio;
  const int e = exponent_of((double)X_SCALE / (sqrt(s) + (double)p.g.eps), ratio);
  const float r = (float)ratio;
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int piece = i * NT + t, row = piece % (SIDE / 8) * 8, col = piece / (SIDE / 8);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[i][q] = __builtin_ldexpf(v[i][q], e);
    if (!p.turn) {
      Q::put(X, col, row, f4_t{v[i][0], v[i][1], v[i][2], v[i][3]});
      Q::put(X, col, row + 4, f4_t{v[i][4], v[i][5], v[i][6], v[i][7]});
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        *reinterpret_cast<_Float16*>(X + Q::at(row + q, col & ~3) + (col & 3) * 2) = (_Float16)v[i][q];
    }
  }
  __syncthreads();
  f4_t x[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int hi = hi0 + 16 * i, lo = lo0 + 16 * j;
      if (p.g.type != RTAT_TYPE_F32) {
        x[i][j] = Q::get(X, lo, hi);  // exact
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int row = p.turn ? lo : hi + q, col = p.turn ? hi + q : lo;
          const bool in = row < p.g.m && col < p.g.n;
          const float g = in ? static_cast<const float*>(p.g.G)[g0 + row + (long)col * p.g.ldg] : 0.0f;
          x[i][j][q] = __builtin_ldexpf(g, e);
        }
      }
    }

  f4_t acc[TM][TN];
#pragma unroll 1
  for (int step = 0; step < p.steps; ++step) {
    const StepFactors& k = p.step[step];
    const float f = step == 0 ? r : 1.0f;
    const bool adds = step < p.steps - 2, last = step == p.steps - 1;
    Q::template multiply<false>(X, X, m0, n0, lane, acc);  // M = X^T X
    const float am = f * f * k.m;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) Q::put(M, lo0 + 16 * j, hi0 + 16 * i, acc[i][j] * am);
    __syncthreads();
    Q::template multiply<false>(M, M, m0, n0, lane, acc);  // P = b M + c M^2 (+ a)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int row = hi0 + 16 * i, col = lo0 + 16 * j;
        f4_t w = acc[i][j] * k.p + Q::get(M, col, row) * k.q;
        if (!adds) {
#pragma unroll
          for (int q = 0; q < 4; ++q) w[q] += row + q == col ? k.diag : 0.0f;
        }
        Q::put(P, col, row, w);
      }
    __syncthreads();
    Q::template multiply<true>(X, P, m0, n0, lane, acc);  // X P (+ a X)
    const float ax = f * k.back, bx = k.a * f;
    __syncthreads();  // X has been read
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        f4_t w = acc[i][j] * ax;
        if (adds) w += x[i][j] * bx;
        x[i][j] = w;
        if (!last) Q::put(X, lo0 + 16 * j, hi0 + 16 * i, w);
      }
    __syncthreads();
  }
  uint16_t* O = p.O + z * p.stride_o;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int hi = hi0 + 16 * i + q, lo = lo0 + 16 * j;
        const int row = p.turn ? lo : hi, col = p.turn ? hi : lo;
        if (row < p.g.m && col < p.g.n)
          O[row + (long)col * p.ldo] = float_to_half(RTAT_TYPE_BF16, x[i][j][q] * (1.0f / X_SCALE));
      }
}

template <int SIDE>
rtat_status_t launch_small(rtat_native_handle* h, const SmallArgs& a, int batch) {
  constexpr int LDS = 3 * Square<SIDE>::BYTES;
  static PerDeviceOnce configured;
  if (!configured(h->device, [&] {
        if (LDS <= 65536) return true;
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(&small_kernel<SIDE>),
                                hipFuncAttributeMaxDynamicSharedMemorySize, LDS) == hipSuccess)
          return true;
        (void)hipGetLastError();
        return false;
      }))
    return RTAT_STATUS_NOT_SUPPORTED;
  hipLaunchKernelGGL((small_kernel<SIDE>), dim3((unsigned)batch), dim3(SMALL_THREADS), LDS, h->stream, a);
  return launch_status();
}

bool is_small(int m, int n) { return m <= 128 && n <= 128; }

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

// One product of a step on matrices of the scratch, of which `used` bytes are the iteration's.
Gemm16 step_product(size_t used, int batch, int m, int n, int k, bool ta, bool tb, const void* A, long lda,
                    long a_stride, const void* B, long ldb, long b_stride, float alpha, void* D,
                    long ldd, long d_stride, int d_type) {
  Gemm16 g = {};
  g.type = RTAT_TYPE_F16;
  g.batch = batch;
  g.scratch_used = used;
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
  g.a_roomy = g.b_roomy = 1;  // padded sides
  g.ep.alpha = alpha;
  g.ep.D = D;
  g.ep.ldd = ldd;
  g.ep.d_stride = d_stride;
  g.ep.d_type = d_type;
  return g;
}

}  // namespace

size_t newton_schulz_workspace_bytes(int m, int n, int batch) {
  if (m <= 0 || n <= 0 || batch <= 0 || is_small(m, n)) return 0;
  // Twelve bytes an element bound the total from above, padding aside; no sum below wraps.
  if (12.0 * batch * ((double)m + 64) * ((double)n + 64) > 0x1p60) return SIZE_MAX;
  return layout_of(m, n, batch).total + 256;
}

rtat_status_t launch_newton_schulz(rtat_native_handle* h, int g_type, int m, int n, int batch,
                                   const void* G, long ldg, long stride_g, int steps,
                                   const float* coeffs, float eps, void* O, long ldo,
                                   long stride_o) {
  NormArgs a = {};
  a.type = g_type;
  a.m = m;
  a.n = n;
  a.G = G;
  a.ldg = ldg;
  a.stride_g = stride_g;
  a.eps = eps;
  if (is_small(m, n)) {
    SmallArgs q = {};
    q.g = a;
    q.turn = m < n;
    q.steps = steps;
    q.O = static_cast<uint16_t*>(O);
    q.ldo = ldo;
    q.stride_o = stride_o;
    step_factors(steps, coeffs, q.step);
    return m <= 64 && n <= 64 ? launch_small<64>(h, q, batch) : launch_small<128>(h, q, batch);
  }
  const size_t bytes = newton_schulz_workspace_bytes(m, n, batch);
  if (bytes == SIZE_MAX) return RTAT_STATUS_ALLOC_FAILED;
  const Layout l = layout_of(m, n, batch);
  unsigned char* ws = static_cast<unsigned char*>(acquire_workspace(h, bytes));
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

  auto blocks_for = [](long pieces) {  // two pieces a thread
    const long b = (pieces + 511) / 512;
    return (int)(b < NORM_BLOCKS ? b : NORM_BLOCKS);
  };
  a.blocks = blocks_for((((long)m + 7) / 8) * n);
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

  StepFactors factors[RTAT_NEWTON_SCHULZ_MAX_STEPS];
  step_factors(steps, coeffs, factors);
  for (int i = 0; i < steps; ++i) {
    const StepFactors& k = factors[i];
    const bool last = i == steps - 1;
    const uint16_t* const x = X[i & 1];
    uint16_t* const y = X[(i + 1) & 1];
    // M = X^T X
    Gemm16 g = step_product(bytes, batch, lp, lp, hp, true, false, x, hp, xs, x, hp, xs, k.m,
                            M, lp, ps, RTAT_TYPE_F16);
    g.tri = 1;
    if (i == 0) {
      g.ep.scale = scale;
      g.ep.r_power = 2;
    }
    st = launch_gemm16(h, g);
    if (st != RTAT_STATUS_SUCCESS) return st;
    // P = b M + c M^2 (+ a)
    g = step_product(bytes, batch, lp, lp, lp, true, false, M, lp, ps, M, lp, ps, k.p, P,
                     lp, ps, RTAT_TYPE_F16);
    g.tri = 1;
    g.ep.beta = k.q;
    g.ep.C = M;
    g.ep.ldc = lp;
    g.ep.c_stride = ps;
    g.ep.c_type = RTAT_TYPE_F16;
    g.ep.diag = k.diag;
    st = launch_gemm16(h, g);
    if (st != RTAT_STATUS_SUCCESS) return st;
    // X = X P (+ a X)
    if (!last) {
      g = step_product(bytes, batch, hp, lp, lp, false, false, x, hp, xs, P, lp, ps, k.back, y, hp,
                       xs, RTAT_TYPE_F16);
      if (adds(i)) {
        const bool f32 = i > 0 || a.F != nullptr;
        g.ep.beta = k.a;
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
      g = step_product(bytes, batch, m, n, lp, true, true, P, lp, ps, x, hp, xs, k.back / X_SCALE,
                       O, ldo, stride_o, RTAT_TYPE_BF16);
    } else {
      g = step_product(bytes, batch, m, n, lp, false, false, x, hp, xs, P, lp, ps,
                       k.back / X_SCALE, O, ldo, stride_o, RTAT_TYPE_BF16);
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
