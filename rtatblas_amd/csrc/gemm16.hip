// Products of 16-bit matrices on the matrix cores (v_mfma_f32_16x16x32_{bf16,f16}) with an
// elementwise epilogue, for the linear layer's forward and backward passes and for the
// Newton-Schulz iteration.  Column-major, D(m x n) = epilogue(op(A) op(B)); f32 accumulation.
//
//   * One workgroup computes a BM x BN tile; K advances BK = 64 elements (128 bytes) at a time
//     through a ring of panels in LDS, or two stages of LDS where operands are not aligned.
//   * Panels keep the orientation they have in memory.  An operand that is contiguous along k
//     ("k-major") lies as rows of 64 k, one 16-byte read per lane and MFMA operand; one that is
//     contiguous along m / n ("mn-major") lies as 64 rows of BM (BN) elements and is read with
//     the transposing LDS load (ds_read_b64_tr_b16: lane i of a group of 16 gets column i of the
//     4 x 16 block that the group addresses), two reads per operand.
//   * Sixteen-byte chunks of a panel row are permuted by an XOR of the row number, which spreads
//     each read over the LDS banks.  Measured clocks per wave instruction, 16 waves of a CU
//     reading: 16 bytes per lane 3.8 with it, 10.3 without; transposing 2.9 with it, 11.0
//     without (row strides of 128 and 512 bytes).
//   * The epilogue turns accumulators into eight neighbouring rows per lane, so that bias,
//     residual, saved activations and results move in 16-byte accesses, by exchanges between
//     lanes; the mirrored half of a symmetric product passes through LDS.
#include <type_traits>

#include "gemm16.h"
#include "gemm16_plan.h"
#include "gemm_plan.h"

namespace rtat_native {

namespace {

struct Gemm16Args {
  int m, n, k, tri;
  int tiles_m, tiles_n, tiles;  // tiles per matrix of the batch
  // slices > 1 (batch 1 only): each tile is computed by that many workgroups, one per slice of the
  // K panels; slice z leaves its raw sums in "matrix" z of D, and join_kernel adds them up.
  int slices;
  const uint16_t* A;
  long lda, a_stride;
  const uint16_t* B;
  long ldb, b_stride;
  // 1: memory behind the last column of a column-wise operand may be read up to a multiple of 8
  // rows, so that a panel with that column needs no guards.
  int a_roomy, b_roomy;
  Epilogue ep;
};

constexpr int BK16 = PANEL16;

template <int BM_, int BN_, int WGM_, int WGN_, int OCC_, int AHEAD_ = 0>
struct Shape16 {
  static constexpr int BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, OCC = OCC_;
  // Panels in a ring of SLOTS, AHEAD of A and of B there or on their way, accumulators of
  // mfma_into; 0: two stages.
  static constexpr int AHEAD = AHEAD_, SLOTS = AHEAD == 3 ? 8 : 5;
  static constexpr bool RING = AHEAD > 0;
  static constexpr int NW = WGM * WGN, NT = 64 * NW;
  static constexpr int WTM = BM / WGM, WTN = BN / WGN;  // wave tile
  static constexpr int TM = WTM / 16, TN = WTN / 16;    // MFMA blocks per wave tile
  static constexpr int STAGE = (BM + BN) * BK16 * 2;    // bytes
  static constexpr int PARK = WTM + 4;                  // floats per parked column
  static constexpr int LDS = RING ? SLOTS * BM * BK16 * 2 : 2 * STAGE;
  static_assert(LDS >= NW * 16 * PARK * 4, "room to park a block column per wave");
};

// A panel of ROWS x 64 elements in LDS, in bytes.
template <bool KMAJOR, int ROWS>
struct Panel16 {
  static constexpr int BYTES = ROWS * BK16 * 2;
  static constexpr int ROWBYTES = KMAJOR ? 128 : ROWS * 2;
  static constexpr int CHUNKS = ROWBYTES / 16;
  // What the chunk index of LDS row r is XORed with.  k-major: eight rows, eight chunks.
  // mn-major: a transposing read takes 32 bytes of each of the rows k = 8 q + 0 .. 3 for two
  // neighbouring q at a time; rows of 256 bytes or more all start at the same bank, 128-byte rows
  // alternate between two.
  __device__ static inline int key(int r) {
    if (KMAJOR) return r & 7;
    if (ROWS >= 128) return 2 * ((r & 3) | ((r >> 1) & 4));
    return 2 * (((r >> 1) & 1) | ((r >> 2) & 2));
  }
  // Chunk c (of the panel, in LDS order) holds elements of LDS row c / CHUNKS, from element
  // 8 * source_chunk(c).
  __device__ static inline int source_chunk(int c) {
    const int r = c / CHUNKS;
    return (c % CHUNKS) ^ key(r);
  }
};

// This lane's place in the MFMA operands of a panel whose wave tile starts at row w0 (a multiple
// of 16): operand `block` (16 rows) of K-step `step` (0 or 1).
template <bool KMAJOR, int ROWS>
struct Frags16 {
  typedef Panel16<KMAJOR, ROWS> P;
  int base;  // bytes
  int flip;  // what the chunk number is XORed with, times 16
  __device__ inline Frags16(int w0, int lane) {
    const int l16 = lane & 15, q = lane >> 4;
    if constexpr (KMAJOR) {
      base = (w0 + l16) * P::ROWBYTES;
      flip = (q ^ P::key(l16)) * 16;
    } else {
      // Lane j of a group addresses 4 elements at row k = 8 q + j / 4 (and + 4), column 4 (j % 4).
      const int k = 8 * q + (l16 >> 2);
      base = k * P::ROWBYTES + (l16 & 1) * 8;
      flip = ((w0 / 8 + ((l16 >> 1) & 1)) ^ P::key(k & 15)) * 16;
    }
  }
  __device__ inline s8_t read(const unsigned char* panel, int block, int step) const {
    if constexpr (KMAJOR) {
      return *reinterpret_cast<const s8_t*>(panel + base + (flip ^ (step * 64)) +
                                            block * 16 * P::ROWBYTES);
    } else {
      typedef __attribute__((address_space(3))) s4_t* lds4_t;
      const unsigned char* at = panel + base + step * 32 * P::ROWBYTES + (flip ^ (block * 32));
      const s4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(at));
      const s4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4_t)(at + 4 * P::ROWBYTES));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // The same with the panel's address in LDS: K-steps and halves (k-major: blocks) are offsets of
  // the instruction, so an address serves several reads.
  __device__ inline s8_t read_at(unsigned panel, int block, int step) const {
    if constexpr (KMAJOR) {
      typedef __attribute__((address_space(3))) const s8_t* lds8_t;
      return ((lds8_t)(uintptr_t)(panel + base + (flip ^ (step * 64))))[block * P::ROWBYTES];
    } else {
      typedef __attribute__((address_space(3))) s4_t* lds4_t;
      const lds4_t at = (lds4_t)(uintptr_t)(panel + base + (flip ^ (block * 32))) + step * 4 * P::ROWBYTES;
      const s4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at);
      const s4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at + P::ROWBYTES / 2);
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// Global -> register -> LDS mover of one panel: any alignment, leading dimension and edge.
// Rows past row_lim repeat the last one (they reach accumulators that are not stored), k past
// k_lim reads as zero.
template <bool KMAJOR, int ROWS, int NT>
struct Mover16 {
  typedef Panel16<KMAJOR, ROWS> P;
  static constexpr int NV = P::BYTES / (16 * NT);
  u4_t r[NV];

  __device__ inline void load(const uint16_t* base, long ld, int row0, int row_lim, int k0,
                              int k_lim, int t) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = i * NT + t, lr = c / P::CHUNKS, e0 = P::source_chunk(c) * 8;
      int row = KMAJOR ? row0 + lr : row0 + e0;
      const int k = KMAJOR ? k0 + e0 : k0 + lr;
      bool whole;
      if constexpr (KMAJOR) {
        row = row < row_lim ? row : row_lim - 1;
        whole = k + 8 <= k_lim;
      } else {
        whole = k < k_lim && row + 8 <= row_lim;
      }
      const uint16_t* at = KMAJOR ? base + (long)row * ld + k : base + (long)k * ld + row;
      if (whole) {
        r[i] = reinterpret_cast<const Loose16*>(at)->v;
      } else {
        s8_t v;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool in = KMAJOR ? k + e < k_lim : (k < k_lim && row + e < row_lim);
          v[e] = in ? (short)at[e] : (short)0;
        }
        r[i] = __builtin_bit_cast(u4_t, v);
      }
    }
  }
  __device__ inline void store(unsigned char* panel, int t) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) *reinterpret_cast<u4_t*>(panel + (i * NT + t) * 16) = r[i];
  }
};

// A block column (16 columns of C) of a wave tile on its way through the wave's own part of LDS:
// parked column by column, taken back as its mirror image.
template <class S>
struct Parked {
  float* park;
  int lane;

  __device__ inline Parked(unsigned char* lds, int wave, int lane_)
      : park(reinterpret_cast<float*>(lds) + wave * 16 * S::PARK), lane(lane_) {}
  // Between a wave's writes and its own reads of what other lanes wrote: LDS keeps the order of a
  // wave's accesses, the compiler has to be told.
  __device__ static inline void turn() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  // Block column j, J <= j < TN: the accumulators must be named by constants.
  template <int J = 0>
  __device__ __forceinline__ void put(int j, const f4_t (&acc)[S::TM][S::TN]) const {
    if (j == J) {
      turn();
#pragma unroll
      for (int i = 0; i < S::TM; ++i) {
        f4_t v = acc[i][J];
        if constexpr (S::RING)
          v = f4_t{mfma_get(acc[i][J][0]), mfma_get(acc[i][J][1]), mfma_get(acc[i][J][2]),
                   mfma_get(acc[i][J][3])};
        *reinterpret_cast<f4_t*>(park + (lane & 15) * S::PARK + 16 * i + 4 * (lane >> 4)) = v;
      }
      turn();
    } else if constexpr (J + 1 < S::TN) {
      put<J + 1>(j, acc);
    }
  }
  // The block column as rows of the mirrored tile: lane pairs take its two halves.
  __device__ inline void get_mirrored(int r0, float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = park[(8 * (lane & 1) + i) * S::PARK + r0 + (lane >> 1)];
  }
};

// Epilogue::scale applied to the factors of matrix z.
__device__ inline void scale_factors(const Epilogue& e, long z, float& alpha, float& beta) {
  if (e.scale == nullptr) return;
  const float r = e.scale[z];
  for (int i = 0; i < e.r_power; ++i) alpha *= r;
  if (e.scale_c) beta *= r;
}

// Two accumulators of neighbouring blocks, 16 rows apart, exchanged between neighbouring groups of
// 16 lanes, so that x and y become the first and second four of eight neighbouring rows of the
// lane's column: rows 16 (q % 2) + 8 (q / 2) .. + 7 of the pair's 32, q = lane / 16.
__device__ inline void pair_up(float& x, float& y) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x),
                                                  __builtin_bit_cast(unsigned, y), false, false);
  const unsigned lo = r[0], hi = r[1];
  x = __builtin_bit_cast(float, lo);
  y = __builtin_bit_cast(float, hi);
}

// Block column J of a wave tile as TM / 2 times eight neighbouring rows, 32 apart.
template <class S, int J>
__device__ __forceinline__ void take_one(const f4_t (&acc)[S::TM][S::TN], float (&v)[S::TM / 2][8]) {
#pragma unroll
  for (int q = 0; q < S::TM / 2; ++q)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if constexpr (S::RING) {
        v[q][r] = mfma_get(acc[2 * q][J][r]);
        v[q][4 + r] = mfma_get(acc[2 * q + 1][J][r]);
      } else {
        v[q][r] = acc[2 * q][J][r];
        v[q][4 + r] = acc[2 * q + 1][J][r];
      }
    }
  asm volatile("; block column %0" : : "n"(J));  // keeps the compiler from merging the copies of this
}
// Block column j, LO <= j < HI: the accumulators must be named by constants.
template <class S, int LO = 0, int HI = S::TN>
__device__ __forceinline__ void take(int j, const f4_t (&acc)[S::TM][S::TN],
                                     float (&v)[S::TM / 2][8]) {
  if constexpr (HI - LO == 1) take_one<S, LO>(acc, v);
  else if (j < (LO + HI) / 2) take<S, LO, (LO + HI) / 2>(j, acc, v);
  else take<S, (LO + HI) / 2, HI>(j, acc, v);
}

// What a block column needs from memory (the residual, or the argument of the activation) is asked
// for one block column ahead.  The accumulators stay in registers: a store instruction covers 64
// neighbouring bytes of 16 columns.  A wave of the largest tile is alone on its SIMD and waits out
// every taken branch, so choices are made once per block column.  EDGE: the wave tile hangs over
// the edge of C, and every access asks how many of its eight rows are inside.
template <class T, class S, bool SLOPE, bool EDGE>
__device__ __forceinline__ void finish_wave(const Epilogue& e, int lane, float alpha, float beta,
                                            int m0, int n0, long z, float* sums_out,
                                            const f4_t (&acc)[S::TM][S::TN]) {
  constexpr int NP = S::TM / 2;
  const int row = m0 + 16 * ((lane >> 4) & 1) + 8 * (lane >> 5), col = n0 + (lane & 15);
  const int left = e.rows - row;  // of the rows from this lane's first on
  const void* in = SLOPE ? (e.act != RTAT_ACT_NONE ? e.aux : nullptr) : e.C;
  const int in_type = SLOPE ? e.aux_type : e.c_type;
  const long ldin = SLOPE ? e.ldaux : e.ldc;
  long in_at = z * (SLOPE ? e.aux_stride : e.c_stride) + row + col * ldin;
  long d_at = z * e.d_stride + row + col * e.ldd;
  long aux_at = z * e.aux_stride + row + col * e.ldaux;
  long copy_at = z * e.copy_stride + row + col * e.ldcopy;
  float each[NP][8];  // the rows' bias, or their sums
#pragma unroll
  for (int q = 0; q < NP; ++q) {
#pragma unroll
    for (int i = 0; i < 8; ++i) each[q][i] = 0.0f;
    if (!SLOPE && e.bias != nullptr) {
      if (EDGE) load8_part(e.bias_type, e.bias, row + 32 * q, left - 32 * q, each[q]);
      else load8(e.bias_type, e.bias, row + 32 * q, each[q]);
    }
  }
  // Sixteen-bit values are asked for ahead; 32-bit ones would take twice the registers.
  const bool ahead = in != nullptr && in_type != RTAT_TYPE_F32;
  auto ask = [&](long at, int c, int q) {
    if (!EDGE) return load16(in, 2 * (at + 32 * q));
    return load16_part(in, at + 32 * q, c < e.cols ? left - 32 * q : 0);
  };
  u4_t next[NP];
#pragma unroll
  for (int q = 0; q < NP; ++q) next[q] = ahead ? ask(in_at, col, q) : u4_t{};
#pragma unroll 1
  for (int j = 0; j < S::TN; ++j) {
    const int here = !EDGE || col + 16 * j < e.cols ? left : 0;
    u4_t now[NP];
#pragma unroll
    for (int q = 0; q < NP; ++q) now[q] = next[q];
    if (ahead && j + 1 < S::TN) {
#pragma unroll
      for (int q = 0; q < NP; ++q) next[q] = ask(in_at + 16 * ldin, col + 16 * (j + 1), q);
    }
    float v[NP][8];
    take<S>(j, acc, v);
#pragma unroll
    for (int q = 0; q < NP; ++q) {
#pragma unroll
      for (int r = 0; r < 4; ++r) pair_up(v[q][r], v[q][4 + r]);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[q][i] = SLOPE ? v[q][i] * alpha : __builtin_fmaf(v[q][i], alpha, each[q][i]);
    }
    if constexpr (SLOPE) {
      if (in != nullptr) act_slopes<NP>(e.act, Half<T>::id, now, v);
#pragma unroll
      for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int i = 0; i < 8; ++i) each[q][i] += !EDGE || here > 0 ? v[q][i] : 0.0f;
    } else {
      if (e.aux != nullptr) {
        store_all<NP, EDGE>(Half<T>::id, e.aux, aux_at, here, v);
        aux_at += 16 * e.ldaux;
      }
      if (e.act != RTAT_ACT_NONE) act_values<NP>(e.act, v);
      if (in != nullptr) {
        if (!ahead) {
#pragma unroll
          for (int q = 0; q < NP; ++q) {
            float c[8];
            if (EDGE) load8_part(RTAT_TYPE_F32, in, in_at + 32 * q, here - 32 * q, c);
            else load8(RTAT_TYPE_F32, in, in_at + 32 * q, c);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[q][i] = __builtin_fmaf(beta, c[i], v[q][i]);
          }
        } else {
          add_scaled<NP>(Half<T>::id, now, beta, v);
        }
      }
      if (e.diag != 0.0f) {
#pragma unroll
        for (int q = 0; q < NP; ++q) add_diagonal(e.diag, row + 32 * q, col + 16 * j, v[q]);
      }
    }
    in_at += 16 * ldin;
    store_all<NP, EDGE>(e.d_type, e.D, d_at, here, v);
    d_at += 16 * e.ldd;
    if (!SLOPE && e.copy != nullptr) {
      store_all<NP, EDGE>(RTAT_TYPE_F16, e.copy, copy_at, here, v);
      copy_at += 16 * e.ldcopy;
    }
  }
  if (SLOPE && sums_out != nullptr) {
    // The sixteen columns add up in a fixed order.
#pragma unroll
    for (int q = 0; q < NP; ++q) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int d = 1; d < 16; d *= 2) each[q][i] += __shfl_xor(each[q][i], d);
      if ((lane & 15) == 0) store8_part(RTAT_TYPE_F32, sums_out, row + 32 * q, left - 32 * q, each[q]);
    }
  }
}

// A wave tile inside C whose epilogue is a factor alone and whose result has the operands' type:
// straight code.
template <class T, class S, int J = 0>
__device__ __forceinline__ void finish_plain(float alpha, uint16_t* at, long ldd,
                                             const f4_t (&acc)[S::TM][S::TN]) {
  constexpr int NP = S::TM / 2;
  float v[NP][8];
  take_one<S, J>(acc, v);
#pragma unroll
  for (int q = 0; q < NP; ++q) {
#pragma unroll
    for (int r = 0; r < 4; ++r) pair_up(v[q][r], v[q][4 + r]);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[q][i] *= alpha;
    store16(at, 64 * q, pack8(Half<T>::id, v[q]));
  }
  __builtin_amdgcn_sched_barrier(0);  // one block column in flight: registers
  if constexpr (J + 1 < S::TN) finish_plain<T, S, J + 1>(alpha, at + 16 * ldd, ldd, acc);
}

template <class T, class S>
__device__ __forceinline__ void finish_tile(const Gemm16Args& p, unsigned char* lds, int tile_m, int tile_n,
                                   long z, int wave, int lane,
                                   const f4_t (&acc)[S::TM][S::TN]) {
  const Epilogue& e = p.ep;
  const int m0 = tile_m * S::BM + (wave % S::WGM) * S::WTM;  // of the wave tile
  const int n0 = tile_n * S::BN + (wave / S::WGM) * S::WTN;
  float alpha = e.alpha, beta = e.beta;
  scale_factors(e, z, alpha, beta);
  // One row of partial sums per wave column.
  float* sums_out =
      e.sums != nullptr ? e.sums + (long)(tile_n * S::WGN + wave / S::WGM) * e.rows : nullptr;
  // The slices of a triangular product are mirrored when they are joined.
  const bool mirror = p.tri != 0 && tile_m != tile_n && p.slices == 1;
  const bool inside = m0 + S::WTM <= e.rows && n0 + S::WTN <= e.cols;
  if (inside && e.plain)
    finish_plain<T, S>(alpha,
                       static_cast<uint16_t*>(e.D) + z * e.d_stride + m0 +
                           16 * ((lane >> 4) & 1) + 8 * (lane >> 5) + (n0 + (lane & 15)) * e.ldd,
                       e.ldd, acc);
  else if (inside && e.slope)
    finish_wave<T, S, true, false>(e, lane, alpha, beta, m0, n0, z, sums_out, acc);
  else if (inside)
    finish_wave<T, S, false, false>(e, lane, alpha, beta, m0, n0, z, sums_out, acc);
  else if (e.slope)
    finish_wave<T, S, true, true>(e, lane, alpha, beta, m0, n0, z, sums_out, acc);
  else
    finish_wave<T, S, false, true>(e, lane, alpha, beta, m0, n0, z, sums_out, acc);
  if (!mirror) return;
  const Parked<S> k(lds, wave, lane);
#pragma unroll 1
  for (int j = 0; j < S::TN; ++j) {
    k.put(j, acc);
#pragma unroll 1
    for (int r0 = 0; r0 < S::WTM; r0 += 32) {
      float v[8];
      k.get_mirrored(r0, v);
      epilogue8(e, alpha, beta, n0 + 16 * j + 8 * (lane & 1), m0 + r0 + (lane >> 1), z, v);
    }
  }
}

// The K range of matrix (or slice) z, and an operand's first element in it.
__device__ inline void k_range(const Gemm16Args& p, long z, int& first, int& len) {
  first = 0;
  len = p.k;
  if (p.slices > 1) {  // panels [z n / slices, (z + 1) n / slices) of the n K panels
    const long n = (p.k + BK16 - 1) / BK16;
    first = (int)(z * n / p.slices) * BK16;
    const int end = (int)((z + 1) * n / p.slices) * BK16;
    len = (end < p.k ? end : p.k) - first;
  }
}
template <bool KMAJOR>
__device__ inline const uint16_t* first_k(const uint16_t* base, long ld, long stride, int slices,
                                          long z, int k) {
  return (slices > 1 ? base : base + z * stride) + (KMAJOR ? (long)k : (long)k * ld);
}

template <class T, class S, bool KA, bool KB>
__global__ __launch_bounds__(S::NT, S::OCC) void gemm16_kernel(Gemm16Args p) {
  constexpr int TM = S::TM, TN = S::TN;
  extern __shared__ __align__(16) unsigned char lds[];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int wm0 = (wave % S::WGM) * S::WTM, wn0 = (wave / S::WGM) * S::WTN;

  const int logical = logical_of_workgroup(blockIdx.x, gridDim.x);
  const long z = logical / p.tiles;
  int tile_m, tile_n;
  tile_of_logical(logical % p.tiles, p.tiles_m, p.tiles_n, p.tri, S::BM, S::BN, tile_m, tile_n);
  const int m0 = tile_m * S::BM, n0 = tile_n * S::BN;
  int k_first, k_len;
  k_range(p, z, k_first, k_len);
  const uint16_t* A = first_k<KA>(p.A, p.lda, p.a_stride, p.slices, z, k_first);
  const uint16_t* B = first_k<KB>(p.B, p.ldb, p.b_stride, p.slices, z, k_first);

  f4_t acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f4_t{0, 0, 0, 0};

  const int panels = (k_len + BK16 - 1) / BK16;
  typedef Panel16<KA, S::BM> PA;
  const Frags16<KA, S::BM> ra(wm0, lane);
  const Frags16<KB, S::BN> rb(wn0, lane);
  Mover16<KA, S::BM, S::NT> ma;
  Mover16<KB, S::BN, S::NT> mb;
  auto load = [&](int kt) {
    ma.load(A, p.lda, m0, p.m, kt * BK16, k_len, t);
    mb.load(B, p.ldb, n0, p.n, kt * BK16, k_len, t);
  };
  auto store = [&](int kt) {
    unsigned char* stage = lds + (kt & 1) * S::STAGE;
    ma.store(stage, t);
    mb.store(stage + PA::BYTES, t);
  };
  if (panels > 0) {
    load(0);
    store(0);
    if (panels > 1) load(1);
  }
  __syncthreads();
  for (int kt = 0; kt < panels; ++kt) {
    const unsigned char* stage = lds + (kt & 1) * S::STAGE;
    if (kt + 1 < panels) store(kt + 1);
    if (kt + 2 < panels) load(kt + 2);
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      s8_t fa[TM], fb[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) fa[i] = ra.read(stage, i, step);
#pragma unroll
      for (int j = 0; j < TN; ++j) fb[j] = rb.read(stage + PA::BYTES, j, step);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = Half<T>::mfma(fa[i], fb[j], acc[i][j]);
    }
    __syncthreads();
  }
  finish_tile<T, S>(p, lds, tile_m, tile_n, z, wave, lane, acc);
}

// Global -> LDS mover of one whole panel (buffer loads that write LDS): nothing passes through
// registers.  Needs 16-byte aligned columns and every k in range; rows over the edge repeat the
// last row (k-major) or the last chunk that starts inside (mn-major: such a chunk may run into
// the next column, so the panel that holds an operand's last column takes Mover16 instead).
template <bool KMAJOR, int ROWS, int NW>
struct Dma16 {
  typedef Panel16<KMAJOR, ROWS> P;
  static constexpr int NI = P::BYTES / (1024 * NW);
  unsigned off[NI];  // bytes from the panel's first element in memory

  __device__ inline void init(long ld, int row0, int row_lim, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int c = (i * NW + wave) * 64 + lane, lr = c / P::CHUNKS, e0 = P::source_chunk(c) * 8;
      if constexpr (KMAJOR) {
        const int row = row0 + lr < row_lim ? lr : row_lim - 1 - row0;
        off[i] = (unsigned)(((long)row * ld + e0) * 2);
      } else {
        const int last = ((row_lim - 1) & ~7) - row0;
        off[i] = (unsigned)(((long)lr * ld + (e0 < last ? e0 : last)) * 2);
      }
    }
  }
  // Instruction i of a panel (`where`: panel_at).  Written in assembly because behind the builtin
  // the compiler waits for every load in flight before each transposing LDS read (the s_nop is the
  // wait state between M0 and a load to LDS); it has no
  // result register, and wait_and_meet is its wait; nothing else here reads M0.
  __device__ inline void issue(int i, u4_t where, unsigned panel, int wave) const {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(panel + (unsigned)(i * NW + wave) * 1024u), "v"(off[i]), "s"(where));
  }
  // Buffer descriptor of panel kt of the operand whose first element of the tile is `base`.
  __device__ static inline u4_t panel_at(const uint16_t* base, long ld, int kt) {
    const uint64_t at =
        reinterpret_cast<uint64_t>(base + (KMAJOR ? (long)kt * BK16 : (long)kt * BK16 * ld));
    return u4_t{(unsigned)at, (unsigned)(at >> 32) & 0xffffu, 0xffffffffu, 0x00020000u};
  }
};
[[maybe_unused]] __device__ inline unsigned lds_address(const unsigned char* p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const unsigned char*)p;
}

// All but the wave's last N loads have arrived and everything it read is in registers; then the
// same of all waves.
template <int N>
[[maybe_unused]] __device__ inline void wait_and_meet() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(N) : "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// The large-tile kernel: 256 x 256 by four waves of 128 x 128, one workgroup per CU.
//   * A wave holds 128 x 128 of C in 256 accumulator registers, which needs the fewest LDS bytes
//     per MFMA (32 reads of 1 KiB for 128 MFMAs of 16 clocks; eight waves of 128 x 64 would ask LDS
//     for 48 in the time it delivers 48).
//   * Panels go straight to LDS, so loads in flight cost no registers.  LDS holds a ring of five
//     32 KiB slots, A and B panels alternating: while panel kt is computed, panel kt + 1 is there
//     or on its way, A of panel kt + 2 is asked for in the first half of kt (the fifth slot) and
//     B in the second half (a slot that kt just left), eight loads in each half.  Loads are so
//     evenly spread that a wave, alone on its SIMD, hardly waits to issue them (all sixteen in one
//     half, into two 64 KiB stages: 8192^3 830 us; bunched at its start 865).
//   * Smaller tiles run the same schedule, two or four workgroups a CU.  Where so few tiles are
//     left that one or two a CU are all there is, a ring of eight slots keeps three panels on
//     their way; a wave is then bound by issuing, and slot numbers modulo a power of two and one
//     address for several reads leave 104 instructions to a panel instead of 150 (us, ring of
//     five / eight: 1024^3 on 64 x 64, TN 7.5 / 6.7, NT 8.7 / 8.2; 2048^3 on 128 x 128, TN
//     21.2 / 18.5).
//   * One barrier per panel, half way through it: by then the second half's operands are in
//     registers, so both slots are free, and of the loads only the last eight may be missing.
//   * Within a half the LDS reads of the next half and the panel loads are spread behind the
//     MFMAs one by one.
template <class T, class S, bool KA, bool KB>
__global__ __launch_bounds__(S::NT, S::OCC) void gemm16_dma_kernel(Gemm16Args p) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass wants the launch stub only
  constexpr int TM = S::TM, TN = S::TN;
  extern __shared__ __align__(16) unsigned char lds[];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm0 = (wave % S::WGM) * S::WTM, wn0 = (wave / S::WGM) * S::WTN;

  const int logical = logical_of_workgroup(blockIdx.x, gridDim.x);
  const long z = logical / p.tiles;
  int tile_m, tile_n;
  tile_of_logical(logical % p.tiles, p.tiles_m, p.tiles_n, p.tri, S::BM, S::BN, tile_m, tile_n);
  const int m0 = tile_m * S::BM, n0 = tile_n * S::BN;
  int k_first, k_len;
  k_range(p, z, k_first, k_len);
  const uint16_t* A = first_k<KA>(p.A, p.lda, p.a_stride, p.slices, z, k_first);
  const uint16_t* B = first_k<KB>(p.B, p.ldb, p.b_stride, p.slices, z, k_first);
  const uint16_t* At = A + (KA ? (long)m0 * p.lda : (long)m0);
  const uint16_t* Bt = B + (KB ? (long)n0 * p.ldb : (long)n0);

  f4_t acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f4_t{0, 0, 0, 0};

  typedef Panel16<KA, S::BM> PA;
  Dma16<KA, S::BM, S::NW> da;
  Dma16<KB, S::BN, S::NW> db;
  da.init(p.lda, m0, p.m, wave, lane);
  db.init(p.ldb, n0, p.n, wave, lane);
  // Panels 0 .. whole - 1 go straight to LDS; a last one may need guards.
  const int panels = (k_len + BK16 - 1) / BK16;
  const bool ragged = k_len % BK16 != 0 ||
                      (k_first + k_len == p.k &&
                       ((!KA && !p.a_roomy && m0 + S::BM > p.m) ||
                        (!KB && !p.b_roomy && n0 + S::BN > p.n)));
  const int whole = panels - (ragged ? 1 : 0);
  // Item 2 kt is A of panel kt, item 2 kt + 1 its B; item x lies in slot x % SLOTS.
  constexpr int AHEAD = S::AHEAD;
  static_assert(AHEAD == 2 || AHEAD == 3, "the waits of the last panels");
  static_assert(S::BM == S::BN && S::LDS >= S::SLOTS * PA::BYTES, "slots of one size");
  auto slot = [&](int item) { return lds + (item % S::SLOTS) * PA::BYTES; };
  auto issue_all = [&](int kt) {
    if (kt < whole) {
      const u4_t pa = da.panel_at(At, p.lda, kt), pb = db.panel_at(Bt, p.ldb, kt);
      const unsigned to_a = lds_address(slot(2 * kt)), to_b = lds_address(slot(2 * kt + 1));
#pragma unroll
      for (int i = 0; i < da.NI; ++i) da.issue(i, pa, to_a, wave);
#pragma unroll
      for (int i = 0; i < db.NI; ++i) db.issue(i, pb, to_b, wave);
    } else {
      {
        Mover16<KA, S::BM, S::NT> ma;
        ma.load(A, p.lda, m0, p.m, kt * BK16, k_len, t);
        ma.store(slot(2 * kt), t);
      }
      Mover16<KB, S::BN, S::NT> mb;
      mb.load(B, p.ldb, n0, p.n, kt * BK16, k_len, t);
      mb.store(slot(2 * kt + 1), t);
    }
  };

  const Frags16<KA, S::BM> ra(wm0, lane);
  const Frags16<KB, S::BN> rb(wn0, lane);
  s8_t fa[2][TM], fb[2][TN];
  // Operand x of a K-step, in the order the MFMAs want them: the first row of A, B, the other rows.
  auto read = [&](const unsigned char* pa, const unsigned char* pb, int step, int x) {
    const int i = x == 0 ? 0 : x - TN;
    if constexpr (S::BM == 256) {  // registers are short there, issue slots are not
      if (x == 0 || x > TN) fa[step][i] = ra.read(pa, i, step);
      else fb[step][x - 1] = rb.read(pb, x - 1, step);
    } else {
      if (x == 0 || x > TN) fa[step][i] = ra.read_at(lds_address(pa), i, step);
      else fb[step][x - 1] = rb.read_at(lds_address(pb), x - 1, step);
    }
  };
  // The MFMAs of one K-step, with read(x), x = 0 .. TM + TN - 1, spread behind the first three
  // quarters of them (as far as there are enough) and load(i), i = 0 .. NLOAD - 1, behind all.
  constexpr int NLOAD = decltype(da)::NI;
  static_assert(NLOAD == decltype(db)::NI && NLOAD <= TM * TN, "a load per MFMA at most");
  auto multiply = [&](int step, auto read_x, auto load_i) {
    constexpr int NMFMA = TM * TN, NREAD = TM + TN;
    constexpr int GAP = 3 * NMFMA >= 4 * NREAD ? 3 * NMFMA / (4 * NREAD) : 1;  // MFMAs to a read
    constexpr int PER = GAP * NREAD <= NMFMA ? 1 : (NREAD + NMFMA - 1) / NMFMA;  // reads at a time
    constexpr int LOAD_GAP = NMFMA / NLOAD > 0 ? NMFMA / NLOAD : 1;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int x = i * TN + j;
        Half<T>::mfma_into(acc[i][j], fa[step][i], fb[step][j]);
        if (x % GAP == 0 && x / GAP * PER < NREAD) {
#pragma unroll
          for (int y = 0; y < PER; ++y)
            if (x / GAP * PER + y < NREAD) read_x(x / GAP * PER + y);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (x % LOAD_GAP == LOAD_GAP / 2 && x / LOAD_GAP < NLOAD) load_i(x / LOAD_GAP);
      }
  };
  auto no_load = [](int) {};

  if (panels > 0) {
    issue_all(0);
#pragma unroll
    for (int i = 1; i < AHEAD; ++i)
      if (i < panels) issue_all(i);
    if (whole >= AHEAD) wait_and_meet<2 * NLOAD * (AHEAD - 1)>();
    else wait_and_meet<0>();
#pragma unroll
    for (int x = 0; x < TM + TN; ++x) read(slot(0), slot(1), 0, x);
  }
  int kt = 0;
  for (; kt < whole - AHEAD; ++kt) {
    const unsigned char *a0 = slot(2 * kt), *b0 = slot(2 * kt + 1);
    const unsigned char *a1 = slot(2 * kt + 2), *b1 = slot(2 * kt + 3);
    const u4_t pa = da.panel_at(At, p.lda, kt + AHEAD), pb = db.panel_at(Bt, p.ldb, kt + AHEAD);
    const unsigned to_a = lds_address(slot(2 * (kt + AHEAD)));
    const unsigned to_b = lds_address(AHEAD == 2 ? a0 : slot(2 * (kt + AHEAD) + 1));
    multiply(0, [&](int x) { read(a0, b0, 1, x); }, [&](int i) { da.issue(i, pa, to_a, wave); });
    wait_and_meet<NLOAD*(2 * AHEAD - 3)>();
    multiply(1, [&](int x) { read(a1, b1, 0, x); }, [&](int i) { db.issue(i, pb, to_b, wave); });
  }
#pragma unroll 1
  for (; kt < panels; ++kt) {
    const unsigned char *a0 = slot(2 * kt), *b0 = slot(2 * kt + 1);
    const unsigned char *a1 = slot(2 * kt + 2), *b1 = slot(2 * kt + 3);
    multiply(0, [&](int x) { read(a0, b0, 1, x); }, no_load);
    if (AHEAD == 3 && kt == whole - 3) wait_and_meet<2 * NLOAD>();  // panel kt + 2 is on its way
    else wait_and_meet<0>();
    if (kt + AHEAD < panels) issue_all(kt + AHEAD);
    multiply(1, [&](int x) { read(a1, b1, 0, x); }, no_load);  // of the last panel: not used
  }
  mfma_settle(acc);
  __syncthreads();
  finish_tile<T, S>(p, lds, tile_m, tile_n, z, wave, lane, acc);
#endif
}

typedef Shape16<256, 256, 2, 2, 1, 2> S256x256;  // loads straight to LDS
typedef Shape16<128, 128, 2, 2, 2, 2> R128x128;
typedef Shape16<128, 128, 2, 2, 1, 3> D128x128;
typedef Shape16<64, 64, 2, 2, 4, 2> R64x64;
typedef Shape16<64, 64, 2, 2, 2, 3> D64x64;
typedef Shape16<128, 128, 2, 2, 2> S128x128;  // any alignment
typedef Shape16<64, 64, 2, 2, 4> S64x64;

// Sums of the slices of a split product, in order, and their epilogue.
constexpr int JOIN_ROWS = 128, JOIN_COLS = 16;  // of C per workgroup
struct JoinArgs {
  Epilogue ep;
  const float* parts;  // slice z: columns of ldp floats, ep.cols of them
  long ldp;
  int slices, tri;
};

__global__ __launch_bounds__(256) void join_kernel(JoinArgs p) {
  __shared__ float part[JOIN_COLS][JOIN_ROWS];
  const int t = threadIdx.x, lr = (t % 16) * 8, lc = t / 16;
  const int row = blockIdx.x * JOIN_ROWS + lr, col = blockIdx.y * JOIN_COLS + lc;
  const Epilogue& e = p.ep;
  // A triangular product leaves the tiles on and below the diagonal.
  if (p.tri != 0 && blockIdx.x < blockIdx.y * JOIN_COLS / JOIN_ROWS) return;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.0f;
  if (row < e.rows && col < e.cols) {
    const float* at = p.parts + row + (long)col * p.ldp;
    const long step = p.ldp * e.cols;
#pragma unroll 4
    for (int z = 0; z < p.slices; ++z) {
      const f4_t* q = reinterpret_cast<const f4_t*>(at + z * step);
      const f4_t lo = q[0], hi = q[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] += lo[i];
        v[4 + i] += hi[i];
      }
    }
  }
  float alpha = e.alpha, beta = e.beta;
  scale_factors(e, 0, alpha, beta);
  const bool mirror = p.tri != 0 && blockIdx.x != blockIdx.y * JOIN_COLS / JOIN_ROWS;
  if (mirror || e.sums != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) part[lc][lr + i] = v[i];
  }
  epilogue8(e, alpha, beta, row, col, 0, v);
  if (mirror) {
    // The same values as sixteen rows of the mirrored columns.
    __syncthreads();
    const int r = t >> 1, c = 8 * (t & 1);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = part[c + i][r];
    epilogue8(e, alpha, beta, blockIdx.y * JOIN_COLS + c, blockIdx.x * JOIN_ROWS + r, 0, v);
  }
  if (e.sums == nullptr) return;  // only gradients have them, and those are never triangular
#pragma unroll
  for (int i = 0; i < 8; ++i) part[lc][lr + i] = v[i];
  __syncthreads();
  if (t < JOIN_ROWS && (int)(blockIdx.x * JOIN_ROWS) + t < e.rows) {
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < JOIN_COLS; ++c) s += part[c][t];
    e.sums[(long)blockIdx.y * e.rows + blockIdx.x * JOIN_ROWS + t] = s;
  }
}

template <class S>
rtat_status_t launch_kernel(rtat_native_handle* h, const Gemm16& g, Gemm16Args p,
                            void (*kern)(Gemm16Args), PerDeviceOnce& configured) {
  if (!configured(h->device, [&] {
        if (S::LDS <= 65536) return true;
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(kern),
                                hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS) == hipSuccess)
          return true;
        (void)hipGetLastError();
        return false;
      }))
    return RTAT_STATUS_NOT_SUPPORTED;
  p.tiles_m = (p.m + S::BM - 1) / S::BM;
  p.tiles_n = (p.n + S::BN - 1) / S::BN;
  const long tiles = p.tri != 0 ? (long)p.tiles_m * (p.tiles_m + 1) / 2 : (long)p.tiles_m * p.tiles_n;
  const long count = tiles * (p.slices > 1 ? p.slices : g.batch);
  if (count > 0x7fffffffL) return RTAT_STATUS_INVALID_VALUE;
  p.tiles = (int)tiles;
  h->sum_rows = p.tiles_n * S::WGN;
  if (p.slices == 1) {
    hipLaunchKernelGGL(kern, dim3((unsigned)count), dim3(S::NT), S::LDS, h->stream, p);
    return launch_status();
  }
  JoinArgs j = {};
  j.ep = p.ep;
  j.parts = static_cast<const float*>(h->split_ws);
  j.ldp = slice_ld16(p.m);
  j.slices = p.slices;
  j.tri = p.tri;
  Epilogue raw = {};
  raw.rows = p.m;
  raw.cols = p.n;
  raw.alpha = 1.0f;
  raw.D = h->split_ws;
  raw.ldd = j.ldp;
  raw.d_stride = j.ldp * p.n;
  raw.d_type = RTAT_TYPE_F32;
  p.ep = raw;
  hipLaunchKernelGGL(kern, dim3((unsigned)count), dim3(S::NT), S::LDS, h->stream, p);
  const rtat_status_t st = launch_status();
  if (st != RTAT_STATUS_SUCCESS) return st;
  static_assert(JOIN_ROWS % JOIN_COLS == 0, "a block of the join lies in one tile row and column");
  const dim3 grid((unsigned)((p.m + JOIN_ROWS - 1) / JOIN_ROWS),
                  (unsigned)((p.n + JOIN_COLS - 1) / JOIN_COLS));
  h->sum_rows = (int)grid.y;
  hipLaunchKernelGGL(join_kernel, grid, dim3(256), 0, h->stream, j);
  return launch_status();
}

template <class T, class S, bool KA, bool KB, bool DMA>
rtat_status_t launch_shape(rtat_native_handle* h, const Gemm16& g, const Gemm16Args& p) {
  static PerDeviceOnce configured;
  if constexpr (DMA) return launch_kernel<S>(h, g, p, &gemm16_dma_kernel<T, S, KA, KB>, configured);
  else return launch_kernel<S>(h, g, p, &gemm16_kernel<T, S, KA, KB>, configured);
}

template <class T, class S, bool DMA>
rtat_status_t launch_ops16(rtat_native_handle* h, const Gemm16& g, const Gemm16Args& p) {
  const bool ka = g.ta, kb = !g.tb;  // contiguous along k
  if (ka && kb) return launch_shape<T, S, true, true, DMA>(h, g, p);
  if (ka) return launch_shape<T, S, true, false, DMA>(h, g, p);
  if (kb) return launch_shape<T, S, false, true, DMA>(h, g, p);
  return launch_shape<T, S, false, false, DMA>(h, g, p);
}

// Whether panels of an operand may go straight to LDS: 16-byte aligned columns, and the farthest
// element of a 256-row panel within 32-bit byte offsets.
bool direct(const void* base, long ld, long stride) {
  return ((reinterpret_cast<uintptr_t>(base) | (uintptr_t)(ld * 2) | (uintptr_t)(stride * 2)) & 15) == 0 &&
         ld < (1L << 23);
}

// Few columns (a single token, or a handful decoded together) of a product whose operands are both
// contiguous along k: the time is that of reading A once.  A workgroup takes sixteen rows, its
// waves a share of k each, straight from memory into registers, eight K-steps in flight; the
// waves' sums meet in LDS.  Nothing is cut across workgroups: 128 of them with sixteen waves each
// read 3.7 TB/s, 512 of them 5.5 to 6.2, and the second launch of a cut costs more than it gives
// until k is long (few_columns16).  Warm calls in a row, A in the memory-side cache (us; 64 x 64 tiles in slices in
// brackets): 8192 x 1 x 2048 6.1 (11.2), 2048 x 13 x 8192 9.0 (13.0), 8192 x 16 x 8192 21.5 (25.1).
constexpr int FEW_DEEP = 8, FEW_WAVES = 16;

template <class T>
__global__ __launch_bounds__(64 * FEW_WAVES) void few_columns_kernel(Gemm16Args p) {
  __shared__ float part[FEW_WAVES][16][17];
  __shared__ float done[16][17];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, waves = blockDim.x >> 6;
  const int l16 = lane & 15, q = lane >> 4, m0 = blockIdx.x * 16;
  // Loads take four neighbouring lanes for the 64 bytes of a row (or column), which memory serves
  // as one; the MFMA wants them sixteen lanes apart, so each operand is handed round the wave.
  const int lr = lane >> 2, lq = lane & 3, from = (4 * l16 + q) * 4;
  const int row = m0 + lr < p.m ? m0 + lr : p.m - 1;
  // Columns that are not there read the first one again: their sums go nowhere.
  const uint16_t* a = p.A + (long)row * p.lda + 8 * lq;
  const uint16_t* b = p.B + (long)(lr < p.n ? lr : 0) * p.ldb + 8 * lq;
  auto hand = [&](s8_t v) {
    typedef int i4_t __attribute__((ext_vector_type(4)));
    const i4_t w = __builtin_bit_cast(i4_t, v);
    i4_t o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __builtin_amdgcn_ds_bpermute(from, w[i]);
    return __builtin_bit_cast(s8_t, o);
  };
  // Whole K-steps of 32 in batches of FEW_DEEP, dealt to the waves in contiguous shares; the steps
  // behind the last batch go to the waves one by one.
  const int steps = p.k / 32, batches = steps / FEW_DEEP, share = (batches + waves - 1) / waves;
  const int first = wave * share, last = first + share < batches ? first + share : batches;
  f4_t acc = {0, 0, 0, 0};
  auto fetch = [&](const uint16_t* at, int step) {
    return *reinterpret_cast<const s8_t*>(at + 32 * (long)step);
  };
  s8_t fa[FEW_DEEP], fb[FEW_DEEP];
  if (first < last) {
#pragma unroll
    for (int u = 0; u < FEW_DEEP; ++u) {
      fa[u] = fetch(a, first * FEW_DEEP + u);
      fb[u] = fetch(b, first * FEW_DEEP + u);
    }
    for (int s = first + 1; s < last; ++s) {
#pragma unroll
      for (int u = 0; u < FEW_DEEP; ++u) {
        acc = Half<T>::mfma(hand(fa[u]), hand(fb[u]), acc);
        fa[u] = fetch(a, s * FEW_DEEP + u);
        fb[u] = fetch(b, s * FEW_DEEP + u);
      }
    }
#pragma unroll
    for (int u = 0; u < FEW_DEEP; ++u) acc = Half<T>::mfma(hand(fa[u]), hand(fb[u]), acc);
  }
  for (int s = batches * FEW_DEEP + wave; s < steps; s += waves)
    acc = Half<T>::mfma(hand(fetch(a, s)), hand(fetch(b, s)), acc);
  if (wave == waves - 1 && p.k % 32 != 0) {  // k is a multiple of 8: a lane's eight are in or out
    s8_t ra = {}, rb = {};
    if (32 * steps + 8 * lq < p.k) {
      ra = fetch(a, steps);
      rb = fetch(b, steps);
    }
    acc = Half<T>::mfma(hand(ra), hand(rb), acc);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) part[wave][l16][4 * q + r] = acc[r];
  __syncthreads();
  const Epilogue& e = p.ep;
  if (t < 256) {
    const int r = t & 15, c = t >> 4;
    float x = 0.0f;
    if (c < p.n && m0 + r < p.m) {
      for (int w = 0; w < waves; ++w) x += part[w][c][r];
      x = epilogue1(e, e.alpha, e.beta, m0 + r, c, 0, x);
    }
    done[c][r] = x;
  }
  if (e.sums == nullptr) return;
  __syncthreads();
  if (t < 16 && m0 + t < p.m) {
    float x = 0.0f;
#pragma unroll
    for (int c = 0; c < 16; ++c) x += done[c][t];
    e.sums[m0 + t] = x;
  }
}

template <class T>
rtat_status_t launch_few_columns(rtat_native_handle* h, const Gemm16Args& p) {
  // Sixteen waves a CU, as far as a workgroup of four to sixteen of them and a batch of K-steps for
  // each allow (8192 x 16 x 8192: eight 22 us, sixteen 30; 1024 x 16 x 1024: four 5.0, eight 5.7).
  const long wgs = ((long)p.m + 15) / 16, cus = h->compute_units > 0 ? h->compute_units : 256;
  long waves = 16 * cus / wgs;
  const long batches = p.k / (32 * FEW_DEEP);
  if (waves > batches) waves = batches;
  waves = waves < 4 ? 4 : (waves > FEW_WAVES ? FEW_WAVES : waves);
  h->sum_rows = 1;
  hipLaunchKernelGGL(few_columns_kernel<T>, dim3((unsigned)((p.m + 15) / 16)),
                     dim3((unsigned)(64 * waves)), 0, h->stream, p);
  return launch_status();
}

// Operands that may not go straight to LDS, laid out anew: columns of `rows` elements, `ldd` apart
// (a multiple of 8) with zeros behind them, and zero columns up to `cols_out`.
struct PackJob {
  const uint16_t* src;
  long ld;
  int rows, cols, cols_out;
  uint16_t* dst;
  long ldd;
};
struct PackArgs {
  PackJob job[2];
};
// A workgroup takes PACK_COLS columns, 32 threads to a column's pieces of eight rows.
constexpr int PACK_COLS = 32;
__global__ __launch_bounds__(256) void pack_kernel(PackArgs p) {
  const PackJob j = p.job[blockIdx.y];
  const int lane = threadIdx.x % 32, first = blockIdx.x * PACK_COLS + threadIdx.x / 32;
  for (int row = (blockIdx.z * 32 + lane) * 8; row < j.ldd; row += gridDim.z * 256) {
    const uint16_t* const at = j.src + (long)first * j.ld + row;
    s8_t v[PACK_COLS / 8];
    // Inside, all loads are on their way before the first is waited for.
    if (row + 8 <= j.rows && first + PACK_COLS - 8 < j.cols) {
#pragma unroll
      for (int c = 0; c < PACK_COLS / 8; ++c)
        v[c] = __builtin_bit_cast(s8_t, load16(at + 8L * c * j.ld, 0));
    } else {
#pragma unroll
      for (int c = 0; c < PACK_COLS / 8; ++c) {
        v[c] = s8_t{};
        if (first + 8 * c < j.cols) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (row + e < j.rows) v[c][e] = (short)at[8L * c * j.ld + e];
        }
      }
    }
#pragma unroll
    for (int c = 0; c < PACK_COLS / 8; ++c)
      if (first + 8 * c < j.cols_out)
        *reinterpret_cast<s8_t*>(j.dst + (first + 8L * c) * j.ldd + row) = v[c];
  }
}

// Copies the operands of a product that are not aligned into scratch, if that pays and the scratch
// is there; true if both operands are direct afterwards.  Worth it when what the faster kernel
// saves (200 against 700 flop per ps where both were measured, around 2 to 13 GFLOP) is more than
// a launch and one trip of the operands through memory.
constexpr size_t PACK_MOST = (size_t)512 << 20;
bool pack_operands(rtat_native_handle* h, const Gemm16& g, Gemm16Args& p, bool direct_a,
                   bool direct_b) {
  if (g.batch != 1 || p.k == 0) return false;
  const bool both = !direct_a && !direct_b;
  const int k_out = both ? (p.k + BK16 - 1) / BK16 * BK16 : p.k;
  auto plan = [&](bool kmajor, const uint16_t* src, long ld, int mn) {
    PackJob j = {};
    j.src = src;
    j.ld = ld;
    j.rows = kmajor ? p.k : mn;
    j.cols = kmajor ? mn : p.k;
    j.cols_out = kmajor ? mn : k_out;
    j.ldd = ((kmajor ? k_out : mn) + 7L) / 8 * 8;
    return j;
  };
  PackJob a = plan(g.ta, p.A, p.lda, p.m), b = plan(!g.tb, p.B, p.ldb, p.n);
  const size_t a_bytes = direct_a ? 0 : ((size_t)a.ldd * a.cols_out * 2 + 255) & ~(size_t)255;
  const size_t b_bytes = direct_b ? 0 : (size_t)b.ldd * b.cols_out * 2;
  const double gflop = 2e-9 * p.m * (double)p.n * p.k;
  if (gflop * (1e3 / 200 - 1e3 / 700) < 5.0 + (double)(a_bytes + b_bytes) * 2 / 4e6) return false;
  const size_t need = g.scratch_used + a_bytes + b_bytes + 256;
  if (need > PACK_MOST) return false;
  uint8_t* ws = static_cast<uint8_t*>(acquire_workspace(h, need));
  if (ws == nullptr) return false;
  ws = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(ws + g.scratch_used) + 255) & ~(uintptr_t)255);
  const Gemm16Args before = p;
  PackArgs q = {};
  int jobs = 0, cols = 0;
  auto add = [&](PackJob& j, uint8_t* to) {
    j.dst = reinterpret_cast<uint16_t*>(to);
    q.job[jobs++] = j;
    cols = j.cols_out > cols ? j.cols_out : cols;
  };
  if (!direct_a) {
    add(a, ws);
    p.A = a.dst;
    p.lda = a.ldd;
    p.a_roomy = 1;
  }
  if (!direct_b) {
    add(b, ws + a_bytes);
    p.B = b.dst;
    p.ldb = b.ldd;
    p.b_roomy = 1;
  }
  if (both) p.k = k_out;
  const long ldd = a.ldd > b.ldd ? a.ldd : b.ldd;
  hipLaunchKernelGGL(pack_kernel,
                     dim3((unsigned)((cols + PACK_COLS - 1) / PACK_COLS), (unsigned)jobs,
                          (unsigned)(ldd < 256 * 16 ? (ldd + 255) / 256 : 16)),
                     dim3(256), 0, h->stream, q);
  if (launch_status() == RTAT_STATUS_SUCCESS) return true;
  p = before;
  return false;
}

template <class T>
rtat_status_t launch_type(rtat_native_handle* h, const Gemm16& g, Gemm16Args p) {
  const bool direct_a = direct(p.A, p.lda, p.a_stride), direct_b = direct(p.B, p.ldb, p.b_stride);
  // A lent workspace means that the library uses no memory of its own: nothing is cut.
  const size_t scratch = h->user_ws == nullptr && h->split_ws != nullptr ? SPLIT_WS_BYTES : 0;
  if (g.ta && !g.tb && direct_a && direct_b && few_columns16(p.m, p.n, p.k, scratch) && g.batch == 1 &&
      g.tri == 0 && g.ep.scale == nullptr)
    return launch_few_columns<T>(h, p);
  const bool ring = (direct_a && direct_b) || pack_operands(h, g, p, direct_a, direct_b);
  const Plan16 plan = plan16(p.m, p.n, p.k, g.batch, g.tri != 0, ring, scratch,
                             h->compute_units > 0 ? h->compute_units : 256);
  p.tri = plan.tri;
  p.slices = plan.slices;
  if (!ring)
    return plan.tile == 128 ? launch_ops16<T, S128x128, false>(h, g, p)
                            : launch_ops16<T, S64x64, false>(h, g, p);
  if (plan.tile == 256) return launch_ops16<T, S256x256, true>(h, g, p);
  // With one 128 x 128 tile a CU, or two of 64 x 64, there is room for the longer ring.
  const long cus = h->compute_units > 0 ? h->compute_units : 256;
  const long side_m = (p.m + plan.tile - 1) / plan.tile, side_n = (p.n + plan.tile - 1) / plan.tile;
  const long tiles = (plan.tri ? side_m * (side_m + 1) / 2 : side_m * side_n) *
                     (plan.slices > 1 ? plan.slices : g.batch);
  if (tiles <= (plan.tile == 128 ? 1 : 2) * cus)
    return plan.tile == 128 ? launch_ops16<T, D128x128, true>(h, g, p)
                            : launch_ops16<T, D64x64, true>(h, g, p);
  return plan.tile == 128 ? launch_ops16<T, R128x128, true>(h, g, p)
                          : launch_ops16<T, R64x64, true>(h, g, p);
}

// out[row] = sum of `count` rows of partial sums, in a fixed order: four threads to a row, each a
// quarter of them.
__global__ __launch_bounds__(256) void sum_rows_kernel(const float* parts, int count, int m,
                                                       float* out) {
  __shared__ float quarter[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.x * 64 + lane;
  float s = 0.0f;
  if (row < m) {
#pragma unroll 8
    for (int i = wave; i < count; i += 4) s += parts[(long)i * m + row];
  }
  quarter[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && row < m)
    out[row] = (quarter[0][lane] + quarter[1][lane]) + (quarter[2][lane] + quarter[3][lane]);
}

}  // namespace

int dact_sum_rows(int n) { return (int)(4 * (((long)n + 63) / 64)); }

rtat_status_t launch_sum_rows(rtat_native_handle* h, const float* parts, int count, int m,
                              float* out) {
  hipLaunchKernelGGL(sum_rows_kernel, dim3((unsigned)((m + 63) / 64)), dim3(256), 0, h->stream,
                     parts, count, m, out);
  return launch_status();
}

rtat_status_t launch_gemm16(rtat_native_handle* h, const Gemm16& g) {
  if (g.m <= 0 || g.n <= 0 || g.batch <= 0) return RTAT_STATUS_SUCCESS;
  Gemm16Args p = {};
  p.m = g.m;
  p.n = g.n;
  p.k = g.k;
  p.tri = g.tri;
  p.slices = 1;
  p.A = static_cast<const uint16_t*>(g.A);
  p.lda = g.lda;
  p.a_stride = g.a_stride;
  p.B = static_cast<const uint16_t*>(g.B);
  p.ldb = g.ldb;
  p.b_stride = g.b_stride;
  p.a_roomy = g.a_roomy;
  p.b_roomy = g.b_roomy;
  p.ep = g.ep;
  const Epilogue& e = g.ep;
  p.ep.plain = !e.slope && e.act == RTAT_ACT_NONE && e.bias == nullptr && e.aux == nullptr &&
               e.C == nullptr && e.copy == nullptr && e.diag == 0.0f && e.d_type == g.type;
  return g.type == RTAT_TYPE_BF16 ? launch_type<__bf16>(h, g, p) : launch_type<_Float16>(h, g, p);
}

}  // namespace rtat_native
