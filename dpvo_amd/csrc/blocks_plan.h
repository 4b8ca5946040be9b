// blocks_plan.h -- which kernel runs a call of the gated blocks and norms, with what tiles, and in how many parts: rules on sizes, types and
// alignment.  Plain C++, no device code: tests/test_blocks.py compiles it to see that the GPU tests reach every choice.
#pragma once
#include <limits.h>
#include <stdint.h>
#include "../../include/dpvo_hip.h"

namespace blk {

constexpr int MAXP = 4;                                  // weight gradients of a call
enum { F_NT = 0, F_NN = 1, F_TN = 2 };                  // (A row, B row) forward; (A row, B col) input gradients; (A col, B col) weight gradients
enum { E_LIN = 0, E_GATE = 1, E_GATE2 = 2, E_DACT = 3 };
// how a product is run: tiles of 128 x 128, 256 x 256 or 64 x 64 (by two waves or four), or few rows with the summed index over the waves (blocks_gemm.h)
enum { T_TILE = 0, T_BIG = 1, T_SMALL = 2, T_TINY = 3, T_FEW = 4 };

inline bool type_ok(int t) { return t == DPVO_F16 || t == DPVO_BF16 || t == DPVO_F32; }
inline int type_size(int t) { return t == DPVO_F32 ? 4 : 2; }
inline bool act_ok(int a) { return a >= DPVO_ACT_IDENTITY && a <= DPVO_ACT_GELU_TANH; }
// row offsets within a tile are 32-bit bytes
inline bool ld_ok(int64_t ld, int64_t width, int size) { return ld >= width && ld <= INT_MAX / (256 * size); }

inline int block_k(int dtype) { return dtype == DPVO_F32 ? 32 : 64; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---- which tiles, and in how many parts the summed index is cut where there are too few of them
struct Plan {
  int kind;
  int64_t splits;
};
inline int tile_size(int kind) { return kind == T_BIG ? 256 : kind == T_SMALL || kind == T_TINY ? 64 : 128; }
// `count(t)`: tiles of t x t; nb: blocks of the summed index; cut: whether parts are possible.
//  - 256 x 256 reads LDS least per product and gives 1127 Tflop/s (bf16, 8192 x 8192 x 4096: 488 us) where 128 x 128 gives 897 (613 us), so a round
//    of the latter (two workgroups on each of 256 compute units) takes 0.62 of a round of the former (one): whichever needs less.  But nothing
//    hides the epilogue of one workgroup alone: with 16 blocks it still wins (73.2 against 86.0 us, 4096 x 4096 x 1024 twice), with 6 it loses
//    (55.8 against 49.5 us, 45312 x 384 x 384 twice); f32 products are bound by the matrix unit and gain nothing.
//  - 128 x 128 wants its two workgroups: at 432 tiles it wins over 64 x 64 (16.6 against 20.4 us, 9216 x 768 x 384), at 256 it loses (20.7 against
//    18.7, 2048 x 2048 x 1024).
//  - Parts: towards two workgroups a compute unit, each with 12 blocks at least (a part costs a tile's write and read in f32, and all of them a
//    launch); dw 384 x 384 over 45312 rows: 45 us in 56 parts, 56 in 64, 59 in 16.  Where that does not fill them, small tiles in parts of 4
//    blocks at least: over 9216 rows 23 us in 21 parts, 25 with large tiles in 16.  Below 16 blocks a second launch costs more than it
//    saves: 333 x 2048 x 768 8.6 us whole, 14.0 in three.
//  - 64 x 64 by four waves where there are few: 1237 x 385 x 882 in f32 24.6 us against 40.5 with two waves, at 864 tiles 13.3 against 11.6.
template <class F> Plan plan(F count, int64_t nb, int dtype, bool cut) {
  const int64_t t = count(128);
  if (dtype != DPVO_F32 && nb >= 16 && ceil_div(count(256), 256) * 100 < ceil_div(t, 512) * 62) return {T_BIG, 1};
  if (t >= 384) return {T_TILE, 1};
  const int small = count(64) >= 640 ? T_SMALL : T_TINY;
  if (!cut || t == 0 || nb < 16) return {small, 1};
  auto parts = [&](int64_t want, int64_t least) {
    const int64_t n = want < nb / least ? want : nb / least;
    return n < 1 ? 1 : n > 64 ? 64 : n;
  };
  const int64_t n = parts(512 / t, 12);
  if (n * t >= 384) return {T_TILE, n};
  return {small, parts(768 / count(64), 4)};
}
inline int64_t tiles(int64_t M, int64_t N, int t) { return ceil_div(M, t) * ceil_div(N, t); }
// A plain projection (no activation, nothing saved) may be cut into parts like a gradient's sum
inline bool linear_cut(const dpvo_gated_linear_t* p) {
  return !p->w_up && p->activation == DPVO_ACT_IDENTITY && !p->save_gate && p->ldy == p->N && (!p->residual || p->ldr == p->N);
}
inline Plan linear_plan(const dpvo_gated_linear_t* p, int epi) {
  const int bk = block_k(p->dtype);
  Plan c = plan([&](int t) { return tiles(p->M, epi == E_GATE ? 2 * p->N : p->N, t); }, ceil_div(p->K, bk) + (epi == E_GATE2 ? ceil_div(p->Kv, bk) : 0),
                p->dtype, linear_cut(p));
  if (epi == E_GATE2 && c.kind == T_BIG) c.kind = T_TILE;      // (two sets of sums do not fit the registers of the largest tile)
  return c;
}
// The few-row kernel's workgroups (64 rows x 16 columns) instead of tiles: up to 16 rows, and wherever they are one to a compute unit at most (f16
// 200 x 1024 x 1024 relu 7.5 against 10.3 us, with 384 of them 12.7 against 10.5); twice as many up to 32 rows, where half of their products are
// for nothing but the weights' bytes count, and for two inputs in f32 (200 x 384 x 384 10.7 against 24.2 us, with 384 of them 18.6 against
// 24.3, with 768 28.1 against 25.0).  Beyond 16 rows not
//  - for 16-bit rows of odd length, whose unaligned pieces the tiles load once and these workgroups again and again (96 x 882 x 385: 14.9 against
//    9.0 us, with 386 columns 7.7 against 8.1; by the length and not the address, so that a result does not depend on where its operands lie),
//  - for long sums that may be cut into parts (f16 96 x 1024 x 4096: 20.1 against 14.8 us, 96 x 768 x 2048 11.5 against 11.8).
// Sums of any length that cannot be cut (a gate, an activation) stay here: M x K x N, one input / two inputs / one product with an activation, against
// tiles, in us: f16 48 x 4096 x 4096 24 / 33 / 18 against 43 / 78 / 41, 96 x 8192 x 1024 45 / 72 / 37 against 80 / 150 / 51, 1000 x 8192 x 256
// 46 / 73 / 38 against 79 / 144 / 75, 1000 x 2048 x 256 15 / 21 / 12 against 17 / 42 / 16; f32 96 x 8192 x 1024 109 / 152 / 74 against 182 / 380 / 178.
inline bool linear_few(const dpvo_gated_linear_t* p, int epi) {
  if (p->M <= 16) return true;
  if (ceil_div(p->N, 16) * ceil_div(p->M, 64) > (p->M <= 32 || (epi == E_GATE2 && p->dtype == DPVO_F32) ? 512 : 256)) return false;
  if (p->dtype != DPVO_F32 && (p->K % 2 || (p->w_up && p->Kv % 2))) return false;
  return !(linear_cut(p) && p->K > 2048);
}
inline int linear_epi(const dpvo_gated_linear_t* p) {
  if (!p->w_up) return E_LIN;
  return p->v == p->x && p->ldv == p->ldx && p->Kv == p->K ? E_GATE : E_GATE2;
}

inline Plan dx_plan(int64_t M, int64_t N, int64_t nb, int dtype, bool cut) { return plan([&](int t) { return tiles(M, N, t); }, nb, dtype, cut); }

inline Plan dw_plan(const dpvo_gated_linear_dw_t* p) {
  return plan([&](int t) {
    int64_t n = 0;
    for (int i = 0; i < p->n; ++i)
      n += tiles(p->N[i], p->K[i], t);
    return n;
  }, ceil_div(p->M, block_k(p->dtype)), p->dtype, true);
}

// How a row of D elements is spread: 8 on each of L lanes, which keeps the backward's arrays of them in registers.  Four or more rows share
// a workgroup where L <= 64 (no barriers there).  RAGGED: D is no multiple of 8.  Rows of more than 4096 elements go to the wide kernels, except
// that the backward of 16-bit ones of up to 8192, in whole pieces and with up to four sums in LDS, still fits 1024 lanes (4096 x 8192: 153 us, wide
// 254; f32 streams spill there: 884 us, wide 350; the forward takes 73 and 76 us, at 4096 x 5120 82 and 74).
struct NormShape { int L; bool ragged; };
constexpr NormShape NORM_SHAPES[] = {{16, false}, {32, false}, {64, false}, {128, false}, {256, false}, {512, false},
                                     {16, true}, {32, true}, {64, true}, {128, true}, {256, true}, {512, true}, {1024, false}};
constexpr int NORM_1024 = 12, NORM_WIDE = 13, NORM_MAX_D = 16384;
inline int norm_sums(const dpvo_residual_norm_t& p, bool shared) {
  return (p.dw != nullptr) + (p.db != nullptr) + (p.dpw != nullptr) + (p.dpb != nullptr) + (shared && p.dgate);
}
inline int norm_shape(const dpvo_residual_norm_t& p, bool back, int sums) {
  if (p.D > 512 * 8) return back && p.D <= 1024 * 8 && p.D % 8 == 0 && p.x_dtype != DPVO_F32 && sums <= 4 ? NORM_1024 : NORM_WIDE;
  int i = p.D % 8 ? 6 : 0;
  while (NORM_SHAPES[i].L * 8 < p.D) ++i;
  return i;
}
inline int norm_slots(int shape) { return shape == NORM_WIDE || NORM_SHAPES[shape].L > 64 ? 1 : 256 / NORM_SHAPES[shape].L; }   // rows at a time in a workgroup

// ---- the norm backward's share of rows
struct NormPlan {
  int sh;
  int64_t groups, rpg, gpb, bpg, blocks;
  bool shared;                                           // gate rows that several rows share
};
inline NormPlan norm_plan(const dpvo_residual_norm_t& p) {
  NormPlan n;
  n.shared = p.f && p.gate && p.groups < p.M;
  n.sh = norm_shape(p, true, norm_sums(p, n.shared));
  n.groups = n.shared ? p.groups : 1;
  n.rpg = n.groups ? p.M / n.groups : 0;
  // 4096 waves, four to a SIMD: enough loads in flight for the memory, few enough that their partial rows stay a few per cent of the traffic
  const int L = n.sh == NORM_WIDE ? 0 : NORM_SHAPES[n.sh].L;
  // (wide rows: rows of 2048 columns' sums, two to four workgroups a compute unit; 4096 x 8192 bf16 221 us in 64 parts, 130 in 128, 138 in 256)
  const int64_t want = n.sh == NORM_WIDE ? 128 : L > 64 ? 4096 / (L / 64) : 1024, rounds = ceil_div(n.rpg, norm_slots(n.sh));
  if (n.groups >= want) {
    n.bpg = 1;
    n.gpb = ceil_div(n.groups, want);
  } else {
    n.gpb = 1;
    n.bpg = n.groups ? want / n.groups : 1;
    if (n.bpg > rounds) n.bpg = rounds < 1 ? 1 : rounds;
  }
  n.blocks = ceil_div(n.groups, n.gpb) * n.bpg;
  return n;
}

}  // namespace blk
