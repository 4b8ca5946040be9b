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
#pragma once
#include "blocks_dev.h"

namespace blk {
namespace {

typedef BLK_T T;
constexpr int KE = Type<T>::KE;
constexpr int BK = 8 * KE;
constexpr bool FINE = sizeof(T) == 4;

template <int BIG> struct Cfg;
template <> struct Cfg<0> { static constexpr int NT = 256, TM = 128, TN = 128, WN = 2, MI = 2; };
template <> struct Cfg<1> { static constexpr int NT = 512, TM = 256, TN = 256, WN = 4, MI = 4; };

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

// One operand's share of a tile: R rows x one block, by NT threads, four 16-byte pieces of registers each
template <int R, int NT, bool TR> struct Stage {
  i4v v[4];
  static_assert(R * 8 == NT * 4, "four chunks per thread");
  // summed index contiguous: chunk c of row (t / 8 + i * NT / 8).  `at(row)`: the row's element offset from the (uniform) base.
  // summed index as rows: thread = (column group of 4, group of KE k)
  uint32_t off[TR ? 1 : 4];
  int c;

  template <class F> __device__ __forceinline__ void init(F at) {
    const int t = threadIdx.x;
    if constexpr (!TR) {
      c = t & 7;
#pragma unroll
      for (int i = 0; i < 4; ++i) off[i] = (uint32_t)((at((t >> 3) + i * (NT / 8)) + c * KE) * (int64_t)sizeof(T));
    } else {
      c = t / (R / 4);
      off[0] = 0;
    }
  }
  // `base`: element (row0, k) of the operand, uniform; nk: elements of the summed index from k on
  __device__ __forceinline__ void load_row(const T* base) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = ld_any<i4v>((const char*)base + off[i]);
  }
  __device__ __forceinline__ void load_row_guard(const T* base, int64_t nk) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      T o[KE];
      raw_guard<KE>((const T*)((const char*)base + off[i]), nk - c * KE, o);
      v[i] = __builtin_bit_cast(i4v, o);
    }
  }
  // `base`: element (k, col0); cols: columns from col0 on
  template <bool GUARD> __device__ __forceinline__ void load_col(const T* base, int64_t ld, int64_t nk, int64_t cols) {
    const int cg = threadIdx.x % (R / 4);
    const T* p = base + (int64_t)c * KE * ld + cg * 4;
    T o[KE][4];
#pragma unroll
    for (int k = 0; k < KE; ++k) {
      if constexpr (GUARD) raw_guard<4>(p + k * ld, c * KE + k < nk ? cols - cg * 4 : 0, o[k]);
      else __builtin_memcpy(o[k], p + k * ld, sizeof(o[k]));
    }
    __builtin_memcpy(v, o, sizeof(v));
  }
  __device__ __forceinline__ void store(char* lds) const {
    if constexpr (!TR) {
      const int r = threadIdx.x >> 3;
#pragma unroll
      for (int i = 0; i < 4; ++i) *(i4v*)(lds + swz(r + i * (NT / 8), c)) = v[i];
    } else {
      const int cg = threadIdx.x % (R / 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        i4v d;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int k = 0; k < 4; ++k) d[k] = v[k][j];
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)                    // rows 2k, 2k+1 of the 8 x 4 piece: dwords 4k + j/2 and 4k + 2 + j/2
            d[k] = (int)__builtin_amdgcn_perm((unsigned)v[k][2 + j / 2], (unsigned)v[k][j / 2], j & 1 ? 0x07060302u : 0x05040100u);
        }
        *(i4v*)(lds + swz(cg * 4 + j, c)) = d;
      }
    }
  }
};

template <int FORM, int EPI, int BIG> __global__ void __launch_bounds__(Cfg<BIG>::NT, 2) gemm_kernel(const GemmArgs args) {
  typedef Cfg<BIG> C;
  constexpr int NT = C::NT, TM = C::TM, TN = C::TN, MI = C::MI, NI = 2;
  constexpr bool TA = FORM == F_TN, TB = FORM != F_NT;
  constexpr bool TWO = EPI == E_GATE2;                   // two accumulators, one after the other
  __shared__ __attribute__((aligned(16))) char lds[2][(TM + TN) * 128];

  // ---- which tile.  Workgroups go to the 8 dies in turn: die x takes the x-th eighth of the tiles, so that tiles that share rows or columns
  // share an L2; within it, 8 row tiles at a time.
  int64_t b;
  {
    const uint32_t n = gridDim.x, q = n / 8, r = n % 8, x = blockIdx.x % 8, i = blockIdx.x / 8;
    b = (int64_t)x * q + (x < r ? x : r) + i;
  }
  int pi = 0;
  for (int i = 1; i < args.n; ++i)
    if (b >= args.p[i].tile0) pi = i;
  const Prob& P = args.p[pi];
  b -= P.tile0;
  const int64_t per = P.tm * P.tn;
  const int split = (int)(b / per);
  b %= per;
  const int64_t g8 = b / (8 * P.tn), in8 = b % (8 * P.tn), gm = P.tm - g8 * 8 < 8 ? P.tm - g8 * 8 : 8;
  const int64_t tmi = g8 * 8 + in8 % gm, tni = in8 / gm;
  constexpr int OUTN = EPI == E_GATE ? TN / 2 : TN;      // columns of C per tile (E_GATE: half of the tile's B rows are the other weight's)
  const int64_t m0 = tmi * TM, n0 = tni * OUTN;
  const int64_t M = P.M, N = P.N;

  Stage<TM, NT, TA> sa;
  Stage<TN, NT, TB> sb;
  const int64_t lda0 = P.lda[0], lda1 = P.lda[1], ldb0 = P.ldb[0], ldb1 = P.ldb[1];
  const int64_t nb0 = P.nb0;
  int cur = -1;                                          // segment whose row offsets are in sa / sb
  auto aim = [&](int seg) {
    const int64_t la = seg ? lda1 : lda0, lb = seg ? ldb1 : ldb0;
    sa.init([&](int r) { const int64_t left = M - 1 - m0; return (r < left ? r : left) * la; });   // rows behind the last: the last (never stored)
    if constexpr (EPI == E_GATE) {
      // rows 64 w .. 64 w + 31 of the tile are the gate's columns of wave column w, the next 32 the other weight's (loaded with its own base)
      sb.init([&](int r) { const int64_t left = N - 1 - n0; const int col = (r >> 6) * 32 + (r & 31); return (col < left ? col : left) * (r & 32 ? ldb1 : ldb0); });
    } else {
      sb.init([&](int r) { const int64_t left = N - 1 - n0; return (r < left ? r : left) * lb; });
    }
    cur = seg;
  };
  const bool inA = !TA || m0 + TM <= M, inB = !TB || n0 + TN <= N;

  auto fetch = [&](int64_t i) {
    const int seg = i >= nb0;
    if (seg != cur) aim(seg);
    const int64_t k = (i - (seg ? nb0 : 0)) * BK, nk = (seg ? P.K[1] : P.K[0]) - k;
    const int64_t la = seg ? lda1 : lda0, lb = seg ? ldb1 : ldb0;
    const T* A = (const T*)(seg ? P.A[1] : P.A[0]);
    const T* B = (const T*)(seg ? P.B[1] : P.B[0]);
    if constexpr (TA) {
      if (nk >= BK && inA) sa.template load_col<false>(A + k * la + m0, la, nk, M - m0);
      else sa.template load_col<true>(A + k * la + m0, la, nk, M - m0);
    } else {
      if (nk >= BK) sa.load_row(A + m0 * la + k);
      else sa.load_row_guard(A + m0 * la + k, nk);
    }
    if constexpr (TB) {
      if (nk >= BK && inB) sb.template load_col<false>(B + k * lb + n0, lb, nk, N - n0);
      else sb.template load_col<true>(B + k * lb + n0, lb, nk, N - n0);
    } else if constexpr (EPI == E_GATE) {
      // chunk i of a thread is row t / 8 + i * NT / 8; NT / 8 is 32 or 64
      const T *W0 = B + n0 * ldb0 + k, *W1 = (const T*)P.B[1] + n0 * ldb1 + k;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = ((int)threadIdx.x >> 3) + i * (NT / 8);
        const T* p = (const T*)((const char*)(r & 32 ? W1 : W0) + sb.off[i]);
        if (nk >= BK) {
          sb.v[i] = ld_any<i4v>(p);
        } else {
          T t[KE];
          raw_guard<KE>(p, nk - sb.c * KE, t);
          sb.v[i] = __builtin_bit_cast(i4v, t);
        }
      }
    } else {
      if (nk >= BK) sb.load_row(B + n0 * lb + k);
      else sb.load_row_guard(B + n0 * lb + k, nk);
    }
  };

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int lr = lane & 31, lh = lane >> 5;

  f16v acc[TWO ? 2 : 1][MI][NI];
#pragma unroll
  for (int a = 0; a < (TWO ? 2 : 1); ++a)
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[a][i][j] = (f16v)(0.f);

  const int64_t ib = P.nb * split / P.splits, ie = P.nb * (split + 1) / P.splits;
  auto multiply = [&](f16v (&c)[MI][NI], const char* buf) {
    const char* la = buf + 0;
    const char* lb = buf + TM * 128;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      i4v fa[MI], fb[NI];
#pragma unroll
      for (int i = 0; i < MI; ++i) fa[i] = *(const i4v*)(la + swz(wm * (MI * 32) + i * 32 + lr, 2 * s + lh));
#pragma unroll
      for (int j = 0; j < NI; ++j) fb[j] = *(const i4v*)(lb + swz(wn * 64 + j * 32 + lr, 2 * s + lh));
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) c[i][j] = mfma(fb[j], fa[i], c[i][j]);
    }
  };
  auto loop = [&](f16v (&c)[MI][NI], int64_t from, int64_t to) {
    for (int64_t i = from; i < to; ++i) {
      if (i + 1 < ie) fetch(i + 1);
      multiply(c, lds[(i - ib) & 1]);
      if (i + 1 < ie) {
        char* d = lds[(i + 1 - ib) & 1];
        sa.store(d);
        sb.store(d + TM * 128);
      }
      __syncthreads();
    }
  };
  if (ib < ie) {
    fetch(ib);
    sa.store(lds[0]);
    sb.store(lds[0] + TM * 128);
  }
  __syncthreads();
  if constexpr (TWO) {
    loop(acc[0], ib, nb0);
    loop(acc[1], nb0, ie);
  } else {
    loop(acc[0], ib, ie);
  }

  // ---- epilogue: 32 rows at a time through the wave's own piece of LDS (the last barrier of the loop freed it), then along rows
  constexpr int PITCH = 68;                              // floats: 272 bytes, so that 8 rows' 16-byte pieces lie in different banks
  float* st = (float*)&lds[0][0] + wave * (32 * PITCH);
  static_assert(sizeof(lds) >= (size_t)(NT / 64) * 32 * PITCH * 4, "epilogue staging");
  constexpr bool PAIR = EPI == E_GATE || EPI == E_GATE2;
  const int act = P.act;
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int q = 0; q < (TWO ? NI : 1); ++q) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const f16v& c = TWO ? acc[j][i][q] : acc[0][i][j];
          f4 v = {c[r4 * 4], c[r4 * 4 + 1], c[r4 * 4 + 2], c[r4 * 4 + 3]};
          *(f4*)(st + lr * PITCH + j * 32 + r4 * 8 + lh * 4) = v;
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      constexpr int LPR = PAIR ? 4 : 8;                  // lanes per row
#pragma unroll 1
      for (int p = 0; p < 32 * LPR / 64; ++p) {
        const int rr = p * (64 / LPR) + lane / LPR, nc = lane % LPR * 8;
        const int64_t m = m0 + wm * (MI * 32) + i * 32 + rr;
        const int64_t n = n0 + (EPI == E_GATE ? wn * 32 : EPI == E_GATE2 ? wn * 64 + q * 32 : wn * 64) + nc;
        if (m >= M || n >= N) continue;
        const int nv = N - n < 8 ? (int)(N - n) : 8;
        float v[8], u[8];
        *(f4*)&v[0] = *(const f4*)(st + rr * PITCH + nc);
        *(f4*)&v[4] = *(const f4*)(st + rr * PITCH + nc + 4);
        if constexpr (PAIR) {
          *(f4*)&u[0] = *(const f4*)(st + rr * PITCH + 32 + nc);
          *(f4*)&u[4] = *(const f4*)(st + rr * PITCH + 32 + nc + 4);
        }
        if constexpr (EPI == E_DACT) {
          if (P.mask) {
            float h[8];
            load_n<T, 8>((const T*)P.mask + m * P.ldmask + n, nv, h);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = h[e] > 0.f ? v[e] : 0.f;
            store_n<T, 8>((T*)P.out0 + m * P.ldo + n, nv, v);
          } else {
            float g[8], y[8];
            load_n<float, 8>(P.save0 + m * N + n, nv, g);
            act_d8<FINE>(act, g, y);
            if (P.save1) {
              load_n<float, 8>(P.save1 + m * N + n, nv, u);
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
          }
        } else if (EPI == E_LIN && P.part) {
          store_n<float, 8>(P.part + ((int64_t)split * M + m) * N + n, nv, v);
        } else {
          float t[8];
          if (P.bias0) {
            load_n<T, 8>((const T*)P.bias0 + n, nv, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += t[e];
          }
          if (P.save0) store_n<float, 8>(P.save0 + m * N + n, nv, v);
          act8<FINE>(act, v);
          if constexpr (PAIR) {
            if (P.bias1) {
              load_n<T, 8>((const T*)P.bias1 + n, nv, t);
#pragma unroll
              for (int e = 0; e < 8; ++e) u[e] += t[e];
            }
            if (P.save1) store_n<float, 8>(P.save1 + m * N + n, nv, u);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= u[e];
          }
          if (P.addend) {
            load_n<T, 8>((const T*)P.addend + m * P.ldadd + n, nv, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += t[e];
          }
          store_n<T, 8>((T*)P.out0 + m * P.ldo + n, nv, v);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
}

template <int FORM, int EPI, int BIG> int go(const GemmArgs& a, int64_t tiles, hipStream_t s) {
  hipLaunchKernelGGL((gemm_kernel<FORM, EPI, BIG>), dim3((unsigned)tiles), dim3(Cfg<BIG>::NT), 0, s, a);
  DPVO_LAUNCH_CHECK();
  return DPVO_OK;
}

}  // namespace

int BLK_ENTRY(const GemmArgs& a, int form, int epi, int big, int64_t tiles, hipStream_t s) {
  if (tiles == 0) return DPVO_OK;
  if (form == F_NT && epi == E_LIN) return go<F_NT, E_LIN, 0>(a, tiles, s);
  if (form == F_NT && epi == E_GATE) return go<F_NT, E_GATE, 0>(a, tiles, s);
  if (form == F_NT && epi == E_GATE2) return go<F_NT, E_GATE2, 0>(a, tiles, s);
  if (form == F_NN && epi == E_LIN) return go<F_NN, E_LIN, 0>(a, tiles, s);
  if (form == F_NN && epi == E_DACT) return go<F_NN, E_DACT, 0>(a, tiles, s);
  if (form == F_TN && epi == E_LIN) return go<F_TN, E_LIN, 0>(a, tiles, s);
  return DPVO_E_UNSUPPORTED;
}

}  // namespace blk
