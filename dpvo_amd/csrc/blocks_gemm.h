// blocks_gemm.h -- the matrix products of the gated blocks for one element type BLK_T (blocks_f16.hip, blocks_bf16.hip, blocks_f32.hip).
//
// A workgroup makes a TM x TN tile of C.  Both operands are staged through LDS as rows of 128 bytes along the summed index (64 16-bit or 32
// f32 elements), double-buffered: the next block's global loads are issued, the present block is multiplied, then the registers are written
// to the other buffer -- one barrier per block.  An operand whose summed index is its ROW (the weight in an input gradient, both operands
// of a weight gradient) is transposed in registers on its way into LDS (8 x 4 elements of 16 bits per thread: sixteen v_perm_b32), so all
// three forms share the multiplication.  16-byte chunk c of row r lies at chunk c ^ (r & 7) ^ ((r >> 3) & 7): reads of 8 or 16
// consecutive rows and the transposed writes touch distinct banks.
//
// The matrix instruction is 32x32 (x16 for 16 bits, x2 for f32), with the N side as its first operand: a lane then holds four consecutive n of
// one row m, and the epilogue passes each wave's 32 x 64 piece through LDS as f32 so that biases, residuals, saved sums and outputs move in
// 16-byte pieces along rows.
//
// What bounds it.  Large sums: the matrix unit and LDS reads -- 8192 x 8192 x 4096 in bf16 488 us (1127 Tflop/s; a plain library product of this
// size 439), f32 4096 x 4096 x 4096 1052 us (131 Tflop/s; 137).  Short sums (K = 384): memory and the epilogue --
// 45312 x 384 x 384, two of them with sigmoid, product, residual and both biases 70 us for 35 MB in, 35 MB of residual and 35 MB out each way through
// LDS, with 1062 tiles on 512 places (the third round is all but empty); saving both sums in f32 adds 139 MB and 30 us.  Few tiles: one
// workgroup's chain of loads, products and epilogue, 8 to 12 us.  Every output needs a bias, an activation, a mask or a second product anyway: with the
// epilogue in the product nothing of size M x N is read back.
#pragma once
#include "blocks_dev.h"

namespace blk {
namespace {

typedef BLK_T T;
constexpr int KE = Type<T>::KE;
constexpr int BK = 8 * KE;
constexpr bool FINE = sizeof(T) == 4;

template <int KIND> struct Cfg;
// NT threads; WN wave columns of 64, WK waves that share a block's steps; MI 32-row pieces of a wave.  DEPTH: blocks whose loads are under way
// (two for the shape that runs alone on its compute unit; for the others two made no difference)
template <> struct Cfg<T_TILE> { static constexpr int NT = 256, TM = 128, TN = 128, WN = 2, WK = 1, MI = 2, DEPTH = 1; };
template <> struct Cfg<T_BIG> { static constexpr int NT = 512, TM = 256, TN = 256, WN = 4, WK = 1, MI = 4, DEPTH = 1; };
template <> struct Cfg<T_SMALL> { static constexpr int NT = 128, TM = 64, TN = 64, WN = 1, WK = 1, MI = 1, DEPTH = 1; };
template <> struct Cfg<T_TINY> { static constexpr int NT = 256, TM = 64, TN = 64, WN = 1, WK = 2, MI = 1, DEPTH = 2; };

__device__ __forceinline__ int swz(int row, int c) { return row * 128 + ((c ^ (row & 7) ^ ((row >> 3) & 7)) << 4); }

__device__ __forceinline__ f16v mfma(i4v a, i4v b, f16v c) {
  if constexpr (sizeof(T) == 4) {
    const f4 x = __builtin_bit_cast(f4, a), y = __builtin_bit_cast(f4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], c, 0, 0, 0);
    return c;
  } else if constexpr (__is_same(T, _Float16)) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  }
}

// nv of N elements at p as raw bits, zeros behind them
template <int N> __device__ __forceinline__ void raw_guard(const T* p, int64_t nv, T (&o)[N]) {
  if (nv >= N) {
    __builtin_memcpy(o, p, sizeof(o));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = i < nv ? p[i] : (T)0.f;
  }
}

// One operand's share of a tile: R rows x one block, by NT threads, NC 16-byte pieces of registers each.
//   summed index contiguous (row): chunk t % 8 of rows t / 8 + i * NT / 8
//   summed index as rows (col): columns NC (t % (R / NC)) .. + NC - 1 of summed indices KE (t / (R / NC)) .. + KE - 1
// Whole blocks are loaded through a buffer descriptor whose base moves on (scalar work only) and per-lane offsets that never change;
// a segment's last blocks through guarded loads.
template <int R, int NT, bool TR> struct Stage {
  static constexpr int NC = R * 8 / NT;
  static_assert(NC == 4 || NC == 2, "pieces per thread");
  typedef i4v Regs[NC];
  static constexpr int RS = NT / 8;                      // rows between a thread's chunks
  uint32_t off[TR ? 1 : NC];                             // bytes from the tile's base
  // where the pieces go in the first buffer: rows 64 apart have their chunks alike
  static constexpr int NL = TR || RS == 16 ? NC : RS == 32 ? 2 : 1;
  uint32_t lds[NL];

  static __device__ __forceinline__ int chunk() { return TR ? (int)threadIdx.x / (R / NC) : (int)threadIdx.x & 7; }
  static __device__ __forceinline__ int row(int i) { return ((int)threadIdx.x >> 3) + i * RS; }
  static __device__ __forceinline__ int col() { return (int)threadIdx.x % (R / NC) * NC; }

  __device__ __forceinline__ void init_lds(uint32_t base) {
#pragma unroll
    for (int i = 0; i < NL; ++i) lds[i] = base + (TR ? swz(col() + i, chunk()) : swz(row(i), chunk()));
  }
  // row: `at(r)`: element offset of tile row r (clamped to the operand); col: `left`: columns from the tile's first on
  template <class F> __device__ __forceinline__ void aim_rows(F at) {
#pragma unroll
    for (int i = 0; i < NC; ++i) off[i] = (uint32_t)((at(row(i)) + chunk() * KE) * (int64_t)sizeof(T));
  }
  __device__ __forceinline__ void aim_cols(int64_t ld, int64_t left) {
    const int64_t last = (left - 1) / NC * NC;           // groups behind the last column: the last group again, not stored
    off[0] = (uint32_t)((chunk() * KE * ld + (col() < last ? col() : last)) * (int64_t)sizeof(T));
  }
  // base: (tile's first row, k), or for the pieces whose bit is set in `other` base1; col: (k, first column).  All scalar.
  __device__ __forceinline__ void load(Regs& v, const T* base, const T* base1, int other, int64_t ld) const {
    if constexpr (!TR) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const __amdgpu_buffer_rsrc_t d = __builtin_amdgcn_make_buffer_rsrc((void*)(other >> i & 1 ? base1 : base), 0, -1, 0x27000);
        v[i] = __builtin_bit_cast(i4v, __builtin_amdgcn_raw_buffer_load_b128(d, off[i], 0, 0));
      }
    } else {
      const __amdgpu_buffer_rsrc_t d = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, -1, 0x27000);
      const uint32_t step = (uint32_t)(ld * sizeof(T));
      constexpr int W = NC * (int)sizeof(T) / 4;         // dwords of a summed index's columns: 4, 2 or 1
      int t[KE * W];
#pragma unroll
      for (int k = 0; k < KE; ++k) {
        if constexpr (W == 4) {
          const i4v x = __builtin_bit_cast(i4v, __builtin_amdgcn_raw_buffer_load_b128(d, off[0], k * step, 0));
#pragma unroll
          for (int w = 0; w < 4; ++w) t[k * 4 + w] = x[w];
        } else if constexpr (W == 2) {
          const i2v x = __builtin_bit_cast(i2v, __builtin_amdgcn_raw_buffer_load_b64(d, off[0], k * step, 0));
          t[k * 2] = x[0];
          t[k * 2 + 1] = x[1];
        } else {
          t[k] = (int)__builtin_amdgcn_raw_buffer_load_b32(d, off[0], k * step, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < NC; ++i) v[i] = i4v{t[i * 4], t[i * 4 + 1], t[i * 4 + 2], t[i * 4 + 3]};
    }
  }
  // the same with zeros for summed indices >= nk (counted from the block's first) and nothing read behind the operand
  __device__ __forceinline__ void load_guard(Regs& v, const T* base, const T* base1, int other, int64_t ld, int64_t nk, int64_t left) const {
    if constexpr (!TR) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        T o[KE];
        raw_guard<KE>((const T*)((const char*)(other >> i & 1 ? base1 : base) + off[i]), nk - chunk() * KE, o);
        v[i] = __builtin_bit_cast(i4v, o);
      }
    } else {
      const T* p = base + (int64_t)chunk() * KE * ld + col();
      T o[KE][NC];
#pragma unroll
      for (int k = 0; k < KE; ++k) raw_guard<NC>(p + k * ld, chunk() * KE + k < nk ? left - col() : 0, o[k]);
      __builtin_memcpy(&v, o, sizeof(v));
    }
  }
  // adds this thread's share of the columns' sums
  static __device__ __forceinline__ void add_cols(const Regs& v, float (&sum)[NC]) {
    T o[KE][NC];
    __builtin_memcpy(o, &v, sizeof(o));
#pragma unroll
    for (int k = 0; k < KE; ++k)
#pragma unroll
      for (int j = 0; j < NC; ++j) sum[j] += (float)o[k][j];
  }
  __device__ __forceinline__ void store(const Regs& v, char* buf, uint32_t flip) const {
    if constexpr (!TR) {
#pragma unroll
      for (int i = 0; i < NC; ++i) *(i4v*)(buf + ((lds[i % NL] + i / NL * NL * RS * 128) ^ flip)) = v[i];
    } else {
      constexpr int W = NC * (int)sizeof(T) / 4;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        i4v d;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (sizeof(T) == 4) {
            d[k] = v[(k * W + j) / 4][(k * W + j) % 4];
          } else {                                       // column j of summed indices 2k and 2k + 1
            const int lo = 2 * k * W + j / 2, hi = lo + W;
            d[k] = (int)__builtin_amdgcn_perm((unsigned)v[hi / 4][hi % 4], (unsigned)v[lo / 4][lo % 4], j & 1 ? 0x07060302u : 0x05040100u);
          }
        }
        *(i4v*)(buf + (lds[j] ^ flip)) = d;
      }
    }
  }
};

template <int FORM, int EPI, int KIND> __global__ void __launch_bounds__(Cfg<KIND>::NT, 2) gemm_kernel(const GemmArgs) {
  typedef Cfg<KIND> C;
  constexpr int NT = C::NT, TM = C::TM, TN = C::TN, MI = C::MI, NI = 2;
  constexpr bool TA = FORM == F_TN, TB = FORM != F_NT;
  constexpr bool TWO = EPI == E_GATE2;                   // two accumulators, one after the other
  constexpr uint32_t HALF = (TM + TN) * 128;             // one buffer; a power of two, so that an XOR turns to the other
  constexpr int PITCH = 68;                              // epilogue: floats of a row of 64; 272 bytes, so that 8 rows' pieces lie in different banks
  constexpr uint32_t STAGING = NT / 64 * 32 * PITCH * 4;
  __shared__ __attribute__((aligned(16))) char lds[2 * HALF > STAGING ? 2 * HALF : STAGING];

  // ---- which tile.  Workgroups go to the 8 dies in turn: die x takes the x-th eighth of the tiles, so that tiles that share rows or columns
  // share an L2; within it, 8 row tiles at a time.
  int64_t b;
  {
    const uint32_t n = gridDim.x, q = n / 8, r = n % 8, x = blockIdx.x % 8, i = blockIdx.x / 8;
    b = (int64_t)x * q + (x < r ? x : r) + i;
  }
  // (the arguments where they lie, by the scalar unit: indexing the parameter itself would copy it to scratch)
  const GemmArgs& all = *(const GemmArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  int pi = 0;
  if constexpr (FORM == F_TN)
    for (int i = 1; i < all.n; ++i)
      if (b >= all.p[i].tile0) pi = i;
  const Prob& P = all.p[pi];
  b -= P.tile0;
  const int64_t per = P.tm * P.tn;
  const int split = (int)(b / per);
  b %= per;
  const int64_t g8 = b / (8 * P.tn), in8 = b % (8 * P.tn), gm = P.tm - g8 * 8 < 8 ? P.tm - g8 * 8 : 8;
  const int64_t tmi = g8 * 8 + in8 % gm, tni = in8 / gm;
  constexpr int OUTN = EPI == E_GATE ? TN / 2 : TN;      // columns of C per tile (E_GATE: half of the tile's B rows are the other weight's)
  const int64_t m0 = tmi * TM, n0 = tni * OUTN;
  const int64_t M = P.M, N = P.N;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wk = wave % C::WK, wn = wave / C::WK % C::WN, wm = wave / (C::WK * C::WN);
  const int lr = lane & 31, lh = lane >> 5;

  // ---- operands
  Stage<TM, NT, TA> sa;
  Stage<TN, NT, TB> sb;
  sa.init_lds(0);
  sb.init_lds(TM * 128);
  const int64_t lda0 = P.lda[0], lda1 = P.lda[1], ldb0 = P.ldb[0], ldb1 = P.ldb[1];
  const int64_t nb0 = P.nb0, K0 = P.K[0], K1 = P.K[1];
  // E_GATE: rows 64 w .. 64 w + 31 of the tile's B are the gate's columns of wave column w, the next 32 the other weight's
  int other = 0;
  if constexpr (EPI == E_GATE)
#pragma unroll
    for (int i = 0; i < sb.NC; ++i) other |= ((wave * 8 + i * (NT / 8)) >> 5 & 1) << i;
  // a tile that hangs over the last column of a col operand: its last group of four may read up to three elements into the rows that follow,
  // which must exist
  const int spare = (TA && m0 + TM > M) || (TB && n0 + TN > N) ? 4 : 0;
  const T *pa = nullptr, *pb = nullptr, *pb1 = nullptr;  // the next block's base
  int64_t la = 0, lb = 0;
  int64_t run = 0;                                       // blocks from `pa`, `pb` on that need no guard
  int cur = -1;                                          // segment that the row offsets are for

  f16v acc[TWO ? 2 : 1][MI][NI];
#pragma unroll
  for (int a = 0; a < (TWO ? 2 : 1); ++a)
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[a][i][j] = (f16v)(0.f);

  // ---- one block: four steps of two chunks.  Row r + 32 has its chunks at c ^ 4 of row r, so four offsets serve every row of a lane
  uint32_t oa[4], ob[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int c = 2 * (C::WK == 1 ? s : s ^ (2 * wk)) + lh;      // WK = 2: wave wk's two steps come first
    oa[s] = swz(wm * (MI * 32) + lr, c);
    ob[s] = TM * 128 + swz(wn * 64 + lr, c);
  }
  // (a wave at its products before one at its loads: 495 against 509 us for the 256-wide tile at 8192 x 8192 x 4096; the smaller ones gain nothing)
  constexpr bool FIRST = KIND == T_BIG;
  auto multiply = [&](f16v (&c)[MI][NI], uint32_t flip) BLK_INLINE {
    if constexpr (FIRST) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int t = 0; t < 4 / C::WK; ++t) {
      i4v fa[MI], fb[NI];
#pragma unroll
      for (int j = 0; j < NI; ++j) fb[j] = *(const i4v*)(lds + ((ob[t ^ (j & 1 ? 2 : 0)] + j * 4096) ^ flip));
#pragma unroll
      for (int i = 0; i < MI; ++i) fa[i] = *(const i4v*)(lds + ((oa[t ^ (i & 1 ? 2 : 0)] + i * 4096) ^ flip));
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) c[i][j] = mfma(fb[j], fa[i], c[i][j]);
    }
    if constexpr (FIRST) __builtin_amdgcn_s_setprio(0);
  };

  const int64_t ib = P.nb * split / P.splits, ie = P.nb * (split + 1) / P.splits;
  // block i into registers
  auto fetch = [&](int64_t i, typename decltype(sa)::Regs& va, typename decltype(sb)::Regs& vb) BLK_INLINE {
    int64_t nk = 0;
    if (run == 0) {                                      // a segment's first block, or one of its last
      const int seg = i >= nb0;
      const int64_t j = i - (seg ? nb0 : 0), k = j * BK, K = seg ? K1 : K0;
      if (seg != cur) {
        cur = seg;
        la = seg ? lda1 : lda0;
        lb = seg ? ldb1 : ldb0;
        // rows behind an operand's last: the last one again, not stored
        if constexpr (TA) sa.aim_cols(la, M - m0);
        else sa.aim_rows([&](int r) BLK_INLINE { const int64_t left = M - 1 - m0; return (r < left ? r : left) * la; });
        if constexpr (TB) sb.aim_cols(lb, N - n0);
        else if constexpr (EPI == E_GATE)
          sb.aim_rows([&](int r) BLK_INLINE { const int64_t left = N - 1 - n0; const int c = (r >> 6) * 32 + (r & 31); return (c < left ? c : left) * (r & 32 ? ldb1 : ldb0); });
        else
          sb.aim_rows([&](int r) BLK_INLINE { const int64_t left = N - 1 - n0; return (r < left ? r : left) * lb; });
      }
      pa = (const T*)(seg ? P.A[1] : P.A[0]) + (TA ? k * la + m0 : m0 * la + k);
      pb = (const T*)(seg ? P.B[1] : P.B[0]) + (TB ? k * lb + n0 : n0 * lb + k);
      if constexpr (EPI == E_GATE) pb1 = (const T*)P.B[1] + n0 * ldb1 + k;
      run = K - spare > 0 ? (K - spare) / BK - j : 0;
      if (run <= 0) {
        run = 0;
        nk = K - k;
      }
    }
    if (run > 0) {
      sa.load(va, pa, pa, 0, la);
      sb.load(vb, pb, pb1, other, lb);
      pa += TA ? BK * la : BK;
      pb += TB ? BK * lb : BK;
      if constexpr (EPI == E_GATE) pb1 += BK;
      --run;
    } else {
      sa.load_guard(va, pa, pa, 0, la, nk, M - m0);
      sb.load_guard(vb, pb, pb1, other, lb, nk, N - n0);
    }
  };
  const bool colsum = FORM == F_TN && P.colsum && tni == 0;
  float cs[sa.NC] = {};
  auto keep = [&](typename decltype(sa)::Regs& va, typename decltype(sb)::Regs& vb, uint32_t flip) BLK_INLINE {
    if constexpr (FORM == F_TN)
      if (colsum) sa.add_cols(va, cs);
    sa.store(va, lds, flip);
    sb.store(vb, lds, flip);
  };
  constexpr int DEPTH = TWO ? 1 : C::DEPTH;              // (two sets of sums leave no room)
  typename decltype(sa)::Regs ra[DEPTH];
  typename decltype(sb)::Regs rb[DEPTH];
  // block i is multiplied from one buffer while block i + 1 goes from registers to the other and block i + DEPTH is on its way to registers
  if constexpr (DEPTH == 1) {
    uint32_t flip = HALF;
#pragma unroll
    for (int h = 0; h < (TWO ? 2 : 1); ++h)
      for (int64_t i = h ? nb0 : ib - 1; i < (TWO && !h ? nb0 : ie); ++i) {
        const bool more = i + 1 < ie;
        if (more) fetch(i + 1, ra[0], rb[0]);
        if (h || i >= ib) multiply(acc[TWO ? h : 0], flip);
        flip ^= HALF;
        if (more) keep(ra[0], rb[0], flip);
        __syncthreads();
      }
  } else {
    for (int64_t i = ib - 2; i < ie; i += 2) {
      if (i + 2 < ie) fetch(i + 2, ra[0], rb[0]);
      if (i >= ib) {
        multiply(acc[0], 0);
        if (i + 1 < ie) keep(ra[1], rb[1], HALF);
        __syncthreads();
      }
      if (i + 1 >= ie) break;
      if (i + 3 < ie) fetch(i + 3, ra[1], rb[1]);
      if (i >= ib) multiply(acc[0], HALF);
      if (i + 2 < ie) keep(ra[0], rb[0], 0);
      __syncthreads();
    }
    __syncthreads();
  }

  // ---- column sums of A (a bias's gradient: the values are in hand, one column of tiles adds them up)
  if constexpr (FORM == F_TN) {
    if (colsum) {
      float* f = (float*)lds;                            // [8][TM]
#pragma unroll
      for (int j = 0; j < sa.NC; ++j) f[sa.chunk() * TM + sa.col() + j] = cs[j];
      __syncthreads();
      for (int c = threadIdx.x; c < TM; c += NT)
        if (m0 + c < M) {
          float v = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) v += f[k * TM + c];
          if (P.part) ((float*)P.colsum)[split * M + m0 + c] = v;
          else ((T*)P.colsum)[m0 + c] = (T)v;
        }
      __syncthreads();
    }
  }

  // Roundings: everything here is f32 up to the stores.  What is stored in T is what the matrix unit takes in T: a hidden product or layer (E_GATE,
  // E_LIN with an activation) as the next product's operand, dG and dU (E_DACT) as those of dx and dw; a bias's gradient sums the same rounded values,
  // so that it is the gradient of the operand that was used.  A second, finer operand would double the products.
  // ---- epilogue: 32 rows at a time through the wave's own piece of LDS (the last barrier of the loop freed it), then along rows.  Where there
  // are two sums, or an activation, a rolled loop does the work (the activations are long); where there is one, what follows it is short and
  // unrolled, and what that needs from memory (a residual, a mask) is requested for all its rows beforehand, so that a piece waits once
  // (8192 x 8192 x 4096: 499 -> 488 us, 4096 x 4096 x 1024: 43.4 -> 39.0; the pairs gain nothing by it).
  float* st = (float*)lds + wave * (32 * PITCH);
  float* const st0 = st - wk * (32 * PITCH);             // of the first of the waves that share the steps
  constexpr bool PAIR = EPI == E_GATE || EPI == E_GATE2;
  constexpr int LPR = PAIR ? 4 : 8, RPP = 64 / LPR;      // lanes per row, rows per pass
  constexpr int NP = 32 / RPP / C::WK;                   // passes of this wave
  const int act = P.act;
  const bool parts = EPI == E_LIN && P.part;
  const int nc = lane % LPR * 8;
  // a pass's row of this lane; a row's sums
  auto row_of = [&](int p) BLK_INLINE { return (p * C::WK + wk) * RPP + lane / LPR; };
  auto sums = [&](float (&o)[8], int rr, int at) BLK_INLINE {
    const float* q = st0 + rr * PITCH + at;
    f4 x = *(const f4*)q, y = *(const f4*)(q + 4);
#pragma unroll
    for (int k = 1; k < C::WK; ++k) {
      x += *(const f4*)(q + k * (32 * PITCH));
      y += *(const f4*)(q + k * (32 * PITCH) + 4);
    }
    *(f4*)&o[0] = x;
    *(f4*)&o[4] = y;
  };
#pragma unroll
  for (int q = 0; q < (TWO ? NI : 1); ++q) {
    const int64_t n = n0 + (EPI == E_GATE ? wn * 32 : EPI == E_GATE2 ? wn * 64 + q * 32 : wn * 64) + nc;
    const int nv = n >= N ? 0 : N - n < 8 ? (int)(N - n) : 8;
    float b0[8] = {}, b1[8] = {};
    if (EPI != E_DACT && !parts) {
      if (P.bias0) load_n<T, 8>((const T*)P.bias0 + n, nv, b0);
      if (PAIR && P.bias1) load_n<T, 8>((const T*)P.bias1 + n, nv, b1);
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int64_t mi = m0 + wm * (MI * 32) + i * 32;
      const T* extra = nullptr;                          // residual, or the mask
      int64_t ldx = 0;
      if constexpr (EPI == E_DACT) {
        extra = (const T*)P.mask;
        ldx = P.ldmask;
      } else if (!parts) {
        extra = (const T*)P.addend;
        ldx = P.ldadd;
      }
      constexpr bool EARLY = !PAIR && (EPI != E_DACT || KIND != T_BIG);   // (the largest tile's products leave it no registers)
      T pre[EARLY ? NP : 1][8];
      if (EARLY && extra) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const int64_t m = mi + row_of(p);
          if (m < M && nv == 8) __builtin_memcpy(pre[p], extra + m * ldx + n, sizeof(pre[p]));
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const f16v& c = TWO ? acc[j][i][q] : acc[0][i][j];
          f4 v = {c[r4 * 4], c[r4 * 4 + 1], c[r4 * 4 + 2], c[r4 * 4 + 3]};
          *(f4*)(st + lr * PITCH + j * 32 + r4 * 8 + lh * 4) = v;
        }
      if constexpr (C::WK == 1) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      } else {
        __syncthreads();                                 // the sums of the waves that share the steps are added as they are read
      }
      // ---- first pass
      const bool first = PAIR || (EPI == E_LIN && !parts && (act != DPVO_ACT_IDENTITY || P.save0)) || (EPI == E_DACT && !P.mask);
      if (first) {
#pragma unroll 1
        for (int p = 0; p < NP; ++p) {
          const int rr = row_of(p);
          const int64_t m = mi + rr;
          if (m >= M || nv == 0) continue;
          float v[8], u[8];
          sums(v, rr, nc);
          if constexpr (EPI == E_DACT) {
            float g[8], y[8];
            load_n<float, 8>(P.save0 + m * N + n, nv, g);
            if (P.save1) load_n<float, 8>(P.save1 + m * N + n, nv, u);
            act_d_n<FINE, true, 8>(act, g, y);
            if (P.save1) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                y[e] *= v[e];
                v[e] *= u[e];
              }
              store_n<T, 8>((T*)P.out1 + m * P.ldo + n, nv, y);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= g[e];
            store_n<T, 8>((T*)P.out0 + m * P.ldo + n, nv, v);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += b0[e];
            if (P.save0) store_n<float, 8>(P.save0 + m * N + n, nv, v);
            act_n<FINE, true, 8>(act, v);
            if constexpr (PAIR) {
              sums(u, rr, 32 + nc);
#pragma unroll
              for (int e = 0; e < 8; ++e) u[e] += b1[e];
              if (P.save1) store_n<float, 8>(P.save1 + m * N + n, nv, u);
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] *= u[e];
            }
            if constexpr (PAIR) {
              if (extra) {
                load_n<T, 8>(extra + m * ldx + n, nv, u);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += u[e];
              }
              store_n<T, 8>((T*)P.out0 + m * P.ldo + n, nv, v);
            } else {
              *(f4*)(st0 + rr * PITCH + nc) = *(const f4*)&v[0];
              *(f4*)(st0 + rr * PITCH + nc + 4) = *(const f4*)&v[4];
            }
          }
        }
      }
      // ---- second pass of one sum (each lane reads back what it wrote itself)
      if (!PAIR && (EPI != E_DACT || P.mask)) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const int rr = row_of(p);
          const int64_t m = mi + rr;
          if (m < M && nv) {
            float v[8];
            if (first) {
              *(f4*)&v[0] = *(const f4*)(st0 + rr * PITCH + nc);
              *(f4*)&v[4] = *(const f4*)(st0 + rr * PITCH + nc + 4);
            } else {
              sums(v, rr, nc);
              if constexpr (EPI == E_LIN)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += b0[e];
            }
            if (parts) {
              store_n<float, 8>(P.part + ((int64_t)split * M + m) * N + n, nv, v);
            } else {
              if (extra) {
                float t[8];
                if (EARLY && nv == 8) {
#pragma unroll
                  for (int e = 0; e < 8; ++e) t[e] = (float)pre[EARLY ? p : 0][e];
                } else {
                  load_n<T, 8>(extra + m * ldx + n, nv, t);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = EPI == E_DACT ? (t[e] <= 0.f ? 0.f : v[e]) : v[e] + t[e];   // (a NaN passes)
              }
              store_n<T, 8>((T*)P.out0 + m * P.ldo + n, nv, v);
            }
          }
        }
      }
      if constexpr (C::WK == 1) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      } else {
        __syncthreads();
      }
    }
  }
}

// ---- few rows: the weights are read once (for 64 rows) and little else counts, so a workgroup takes 16 columns of C and its W waves share the
// summed index; each lane loads its 16 bytes of a weight row straight into the matrix instruction's operand (16x16, the weight's 16 rows on
// the first side), a batch of loads at a time.  The waves' sums meet in LDS and are added in the waves' order.
// One row of bf16, 2 x 4096 x 1024 and 1024 x 4096: 5.6 us (17 MB at 3.0 TB/s) and 7.8 us (8 MB: 64 workgroups only, each a chain of 8 KB of loads per wave).
__device__ __forceinline__ f4 mfma16(i4v a, i4v b, f4 c) {
  if constexpr (sizeof(T) == 4) {
    const f4 x = __builtin_bit_cast(f4, a), y = __builtin_bit_cast(f4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], c, 0, 0, 0);
    return c;
  } else if constexpr (__is_same(T, _Float16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  }
}

template <int MT, int W, int NW> struct Few {
  static constexpr int KS = 4 * KE, UN = MT == 1 ? 8 : 4;
  const T* x[MT];
  const T* w[NW];
  f4 (*acc)[MT];                                         // [NW][MT]

  // steps s0 .. s0 + UN - 1, of which those from `lim` on count as zeros
  template <bool ALL> __device__ __forceinline__ void batch(int64_t s0, int64_t lim) {
    i4v fx[UN][MT], fw[UN][NW];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int64_t k = (ALL || s0 + u < lim ? s0 + u : lim - 1) * KS;
#pragma unroll
      for (int j = 0; j < NW; ++j) fw[u][j] = ld_any<i4v>(w[j] + k);
#pragma unroll
      for (int i = 0; i < MT; ++i) fx[u][i] = ld_any<i4v>(x[i] + k);
    }
    __builtin_amdgcn_sched_barrier(0);                   // all loads of the batch before the first product
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (!ALL && s0 + u >= lim) break;                  // (uniform)
#pragma unroll
      for (int j = 0; j < NW; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = mfma16(fw[u][j], fx[u][i], acc[j][i]);
    }
  }
  __device__ __forceinline__ void run(int64_t K, int wave) {
    const int lq = (threadIdx.x & 63) >> 4;
    const int64_t steps = (K + KS - 1) / KS, full = K / KS;
    const int64_t from = steps * wave / W, to = steps * (wave + 1) / W, lim = to < full ? to : full;
    int64_t s = from;
    for (; s + UN <= lim; s += UN) batch<true>(s, lim);
    if (s < lim) batch<false>(s, lim);
    if (to > full && to > from) {                        // the last, partial step
      const int64_t k = full * KS, nk = K - k - lq * KE;
      T o[KE];
      i4v fx[MT], fw[NW];
#pragma unroll
      for (int j = 0; j < NW; ++j) { raw_guard<KE>(w[j] + k, nk, o); fw[j] = __builtin_bit_cast(i4v, o); }
#pragma unroll
      for (int i = 0; i < MT; ++i) { raw_guard<KE>(x[i] + k, nk, o); fx[i] = __builtin_bit_cast(i4v, o); }
#pragma unroll
      for (int j = 0; j < NW; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = mfma16(fw[j], fx[i], acc[j][i]);
    }
  }
};

template <int EPI, int MT, int W> __global__ void __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(W == 16 ? 4 : 2, W == 16 ? 4 : 3))) few_kernel(const GemmArgs args) {
  constexpr int NA = EPI == E_LIN ? 1 : 2;
  __shared__ f4 red[W][NA][MT][64];
  const Prob& P = args.p[0];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lq = lane >> 4;
  const int64_t M = P.M, N = P.N, n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * (16 * MT);
  const int64_t wr = n0 + lr < N ? n0 + lr : N - 1;      // columns behind N, rows behind M: the last again, not stored
  f4 acc[NA][MT];
#pragma unroll
  for (int j = 0; j < NA; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[j][i] = f4{0.f, 0.f, 0.f, 0.f};
  auto rows = [&](const T* (&x)[MT], int seg) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int64_t m = m0 + i * 16 + lr < M ? m0 + i * 16 + lr : M - 1;
      x[i] = (const T*)P.A[seg] + m * P.lda[seg] + lq * KE;
    }
  };
  const T* w0 = (const T*)P.B[0] + wr * P.ldb[0] + lq * KE;
  const T* w1 = NA == 2 ? (const T*)P.B[1] + wr * P.ldb[1] + lq * KE : nullptr;
  if constexpr (EPI == E_GATE) {
    Few<MT, W, 2> f;
    rows(f.x, 0);
    f.w[0] = w0;
    f.w[1] = w1;
    f.acc = acc;
    f.run(P.K[0], wave);
  } else {
#pragma unroll
    for (int j = 0; j < NA; ++j) {
      Few<MT, W, 1> f;
      rows(f.x, j);
      f.w[0] = j ? w1 : w0;
      f.acc = acc + j;
      f.run(P.K[j], wave);
    }
  }
#pragma unroll
  for (int j = 0; j < NA; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) red[wave][j][i][lane] = acc[j][i];
  __syncthreads();
  for (int q = threadIdx.x; q < MT * 64; q += 64 * W) {
    const int i = q >> 6, l = q & 63;
    const int64_t m = m0 + i * 16 + (l & 15), n = n0 + (l >> 4) * 4;
    if (m >= M || n >= N) continue;
    const int nv = N - n < 4 ? (int)(N - n) : 4;
    float v[NA][4], t[4];
#pragma unroll
    for (int j = 0; j < NA; ++j) {
      f4 s = red[0][j][i][l];
#pragma unroll
      for (int k = 1; k < W; ++k) s += red[k][j][i][l];
      const T* bias = (const T*)(j ? P.bias1 : P.bias0);
      if (bias) load_n<T, 4>(bias + n, nv, t);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = bias ? s[e] + t[e] : s[e];
      float* save = j ? P.save1 : P.save0;
      if (save) store_n<float, 4>(save + m * N + n, nv, v[j]);
    }
    act_n<FINE, true, 4>(P.act, v[0]);
    if constexpr (NA == 2) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[0][e] *= v[1][e];
    }
    if (P.addend) {
      load_n<T, 4>((const T*)P.addend + m * P.ldadd + n, nv, t);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[0][e] += t[e];
    }
    store_n<T, 4>((T*)P.out0 + m * P.ldo + n, nv, v[0]);
  }
}

template <int EPI> int few(const GemmArgs& a, int64_t blocks, hipStream_t s) {
  const Prob& p = a.p[0];
  const int64_t K = p.K[0] > p.K[1] ? p.K[0] : p.K[1];
  // 16 waves where 4 would each have more than one batch of eight steps to wait for
  if (p.M > 16) hipLaunchKernelGGL((few_kernel<EPI, 4, 8>), dim3((unsigned)blocks, (unsigned)cdiv64(p.M, 64)), dim3(512), 0, s, a);
  else if (K > 4 * 8 * 4 * KE) hipLaunchKernelGGL((few_kernel<EPI, 1, 16>), dim3((unsigned)blocks), dim3(1024), 0, s, a);
  else hipLaunchKernelGGL((few_kernel<EPI, 1, 4>), dim3((unsigned)blocks), dim3(256), 0, s, a);
  DPVO_LAUNCH_CHECK();
  return DPVO_OK;
}

template <int FORM, int EPI, int KIND> int go(const GemmArgs& a, int64_t tiles, hipStream_t s) {
  hipLaunchKernelGGL((gemm_kernel<FORM, EPI, KIND>), dim3((unsigned)tiles), dim3(Cfg<KIND>::NT), 0, s, a);
  DPVO_LAUNCH_CHECK();
  return DPVO_OK;
}

}  // namespace

int BLK_ENTRY(const GemmArgs& a, int form, int epi, int kind, int64_t tiles, hipStream_t s) {
  if (tiles == 0) return DPVO_OK;
  if (kind == T_FEW) return epi == E_LIN ? few<E_LIN>(a, tiles, s) : epi == E_GATE ? few<E_GATE>(a, tiles, s) : few<E_GATE2>(a, tiles, s);
  // (256 x 256 is never chosen for f32, nor for two inputs: not built)
#define BLK_GO(F, E) if (form == F && epi == E) switch (kind) { \
    case T_BIG: if constexpr (sizeof(T) == 2 && E != E_GATE2) return go<F, E, T_BIG>(a, tiles, s); else return DPVO_E_UNSUPPORTED; \
    case T_SMALL: return go<F, E, T_SMALL>(a, tiles, s); \
    case T_TINY: return go<F, E, T_TINY>(a, tiles, s); \
    default: return go<F, E, T_TILE>(a, tiles, s); }
  BLK_GO(F_NT, E_LIN)
  BLK_GO(F_NT, E_GATE)
  BLK_GO(F_NT, E_GATE2)
  BLK_GO(F_NN, E_LIN)
  BLK_GO(F_NN, E_DACT)
  BLK_GO(F_TN, E_LIN)
#undef BLK_GO
  return DPVO_E_UNSUPPORTED;
}

}  // namespace blk
