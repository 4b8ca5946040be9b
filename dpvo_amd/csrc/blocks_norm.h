// blocks_norm.h -- the norms around a block, for one pair of element types: NX of the residual stream (x, s and their gradients), NB of the
// branch (f, gate and their gradients); h and its gradient are either.
//
//   p = post(f)                      layer: (f - mean) / sqrt(var + eps) * pw + pb,  rms: f / sqrt(mean f^2 + eps) * pw + pb, or f itself
//   s = x + scale * act(gate) * p    written once, rounded to NX
//   h = norm(s)                      of the unrounded s
//
// and backward, with s recomputed from x, f and gate (the same bytes as reading a stored s, and exact):
//   dy = ds + J_norm(s)^T dh;  dx = dy;  q = scale * dy;  dgate = q * p * act'(gate);  dp = q * act(gate);  df = J_post(f)^T dp
//   J^T d = r (d w - mean(d w) - xhat mean(d w xhat))   (rms: without the first mean), with xhat the normalised row and r its factor
//
// A row lives in the registers of L lanes, V pieces of E elements each, so every tensor is read once and statistics are two-pass in f32 at no
// traffic; the next row's loads are under way while a row is computed.  Nothing but memory bounds these kernels.  Gradients of what all rows
// (of a group) share are summed in LDS over a workgroup's rows, then over its row slots, then over workgroups by a second launch: no atomics, the order is fixed.
#pragma once
#include "blocks_dev.h"

namespace blk {

struct NormArgs {
  dpvo_residual_norm_t p;
  uint32_t rows_per_gate;                                // rows that share a gate row
  // backward: a workgroup makes `gpb` whole groups of `rpg` rows, or (bpg > 1) one of the bpg parts of one group
  int64_t groups, rpg, gpb, bpg;
  int shared;                                            // ... where the groups are those of the gate's rows
  float *part_gate, *part_w, *part_b, *part_pw, *part_pb;   // partial sums, a row of D each
};

// How a row of D elements is spread: V pieces of E on each of L lanes, at most 16 elements a lane so that the backward's arrays of them stay in
// registers.  Four or more rows share a workgroup where L <= 64 (no barriers there).  Pieces of 8 where D is a multiple (a piece then exists or not as a whole, and
// no load needs a guard), single elements for other D.
struct NormShape { int L, V, E; };
constexpr NormShape NORM_SHAPES[] = {{16, 1, 8}, {32, 1, 8}, {64, 1, 8}, {128, 1, 8}, {256, 1, 8}, {512, 1, 8}, {1024, 1, 8}, {1024, 2, 8},
                                     {32, 8, 1}, {128, 8, 1}, {512, 8, 1}, {1024, 16, 1}};
constexpr int NORM_MAX_D = 16384;
inline int norm_shape(int D) {
  int i = 0;
  while (D % NORM_SHAPES[i].E || NORM_SHAPES[i].L * NORM_SHAPES[i].V * NORM_SHAPES[i].E < D) ++i;
  return i;
}
inline int norm_slots(int shape) { return NORM_SHAPES[shape].L > 64 ? 1 : 256 / NORM_SHAPES[shape].L; }

int norm_f16(const NormArgs& a, int shape, bool back, int64_t blocks, hipStream_t st);     // branch types; stream: the same or f32
int norm_bf16(const NormArgs& a, int shape, bool back, int64_t blocks, hipStream_t st);
int norm_f32(const NormArgs& a, int shape, bool back, int64_t blocks, hipStream_t st);

namespace {

template <int E> __device__ __forceinline__ void param_n(const void* p, int type, int64_t i, float (&o)[E]) {
  if (type == DPVO_F32) load_n<float, E>((const float*)p + i, E, o);
  else if (type == DPVO_F16) load_n<_Float16, E>((const _Float16*)p + i, E, o);
  else load_n<__bf16, E>((const __bf16*)p + i, E, o);
}

// Sum over L lanes (16, 32 or 64, aligned), in all of them: four DPP steps within 16 lanes, then the halves swapped.  No LDS permutes: their
// latency, six in a row and several sums to a row, was most of the time of a row.
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int L> __device__ __forceinline__ float lane_sum(float v) {
  v = dpp_add<0xB1>(v);                                  // quad_perm 1 0 3 2
  v = dpp_add<0x4E>(v);                                  // quad_perm 2 3 0 1
  v = dpp_add<0x141>(v);                                 // row_half_mirror
  v = dpp_add<0x140>(v);                                 // row_mirror
  if constexpr (L >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
  }
  if constexpr (L >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    v = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
  }
  return v;
}

template <int L> constexpr int threads() { return L > 64 ? L : 256; }

// The lanes of a row
template <int L, int V, int E, bool FINE> struct Row {
  static constexpr int P = V * E, PIECE = E;             // elements of a lane, of a piece
  static constexpr int SLOTS = threads<L>() / L;         // rows at a time in a workgroup
  static constexpr int WPR = L > 64 ? L / 64 : 1;        // waves per row
  int lane, slot, D;
  float* red;                                            // [2][2][WPR] scratch for sums over waves
  int flip = 0;
  float inv;                                             // 1 / D

  __device__ __forceinline__ Row(int D_, float* red_)
      : lane(SLOTS == 1 ? threadIdx.x : threadIdx.x % L),
        slot(SLOTS == 1 ? 0 : L == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : threadIdx.x / L),   // (scalar where it can be)
        D(D_), red(red_), inv(1.f / (float)D_) {}
  __device__ __forceinline__ int col(int i) const { return (lane + i * L) * E; }
  __device__ __forceinline__ bool has(int i) const { return col(i) < D; }      // (D is a multiple of E)
  // over the row's lanes, two sums at once.  Consecutive calls use the two halves of the scratch in turn, so one barrier each is enough.
  __device__ __forceinline__ void sum(float& v, float& u) {
    v = lane_sum<L < 64 ? L : 64>(v);
    u = lane_sum<L < 64 ? L : 64>(u);
    if constexpr (L > 64) {
      flip ^= 2 * WPR;
      if ((threadIdx.x & 63) == 0) {
        red[flip + lane / 64] = v;
        red[flip + WPR + lane / 64] = u;
      }
      __syncthreads();
      v = u = 0.f;
#pragma unroll
      for (int i = 0; i < WPR; ++i) {
        v += red[flip + i];
        u += red[flip + WPR + i];
      }
    }
  }
  __device__ __forceinline__ float sum(float v) {
    float u = 0.f;
    sum(v, u);
    return v;
  }
  template <class T> __device__ __forceinline__ void store(T* p, const float (&v)[P]) const {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (has(i)) store_n<T, E>(p + col(i), E, *(const float(*)[E])(v + i * E));
  }
  __device__ __forceinline__ void param(const void* p, int type, float none, float (&o)[P]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int e = 0; e < E; ++e) o[i * E + e] = none;
      if (p && has(i)) param_n<E>(p, type, col(i), *(float(*)[E])(o + i * E));
    }
  }
  // v -> its normalised row (before weights); returns the row's factor.  Elements behind D stay 0.
  __device__ __forceinline__ float normalise(float (&v)[P], int kind, float eps) {
    float m = 0.f;
    if (kind == DPVO_NORM_LAYER) {
#pragma unroll
      for (int e = 0; e < P; ++e) m += v[e];
      m = sum(m) * inv;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const bool in = has(i);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float& x = v[i * E + e];
        x = in ? x - m : 0.f;
        q += x * x;
      }
    }
    q = sum(q) * inv + eps;
    const float r = FINE ? 1.f / sqrtf(q) : __builtin_amdgcn_rsqf(q);   // (rsq: one unit in the last place of f32)
#pragma unroll
    for (int e = 0; e < P; ++e) v[e] *= r;
    return r;
  }
  // d (gradient behind the weights, 0 behind D) -> gradient of the row; xh: the normalised row
  __device__ __forceinline__ void back(float (&d)[P], const float (&xh)[P], float r, int kind) {
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int e = 0; e < P; ++e) {
      a += d[e];
      b += d[e] * xh[e];
    }
    sum(a, b);
    a = kind == DPVO_NORM_LAYER ? a * inv : 0.f;
    b *= inv;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const bool in = has(i);                            // (behind D the mean alone would be left, and reach the next sum)
#pragma unroll
      for (int e = i * E; e < (i + 1) * E; ++e) d[e] = in ? r * (d[e] - a - xh[e] * b) : 0.f;
    }
  }
};

// A lane's elements as they are stored
template <class T, int P> struct Raw { T v[P]; };
template <class T, class R> __device__ __forceinline__ void load_raw(const R& row, const T* p, Raw<T, R::P>& o) {
  constexpr int E = R::PIECE;
#pragma unroll
  for (int i = 0; i < R::P / E; ++i) {
    if (row.has(i)) {
      __builtin_memcpy(o.v + i * E, p + row.col(i), sizeof(T) * E);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) o.v[i * E + e] = (T)0.f;
    }
  }
}
template <class T, int P> __device__ __forceinline__ void to_f32(const Raw<T, P>& r, float (&o)[P]) {
#pragma unroll
  for (int e = 0; e < P; ++e) o[e] = (float)r.v[e];
}

template <class NX, class NB, int L, int V, int E> __global__ void __launch_bounds__(threads<L>()) norm_kernel(const NormArgs a) {
  typedef Row<L, V, E, sizeof(NX) == 4> R;
  constexpr int P = R::P;
  __shared__ float red[4 * R::WPR];
  const dpvo_residual_norm_t& p = a.p;
  R row(p.D, red);
  float w[P], b[P], pw[P], pb[P];
  row.param(p.w, p.w_dtype, 1.f, w);
  row.param(p.b, p.w_dtype, 0.f, b);
  row.param(p.pw, p.w_dtype, 1.f, pw);
  row.param(p.pb, p.w_dtype, 0.f, pb);
  const int64_t step = (int64_t)gridDim.x * R::SLOTS;
  int64_t m = (int64_t)blockIdx.x * R::SLOTS + row.slot;
  Raw<NX, P> rx;
  Raw<NB, P> rf, rg;
  auto fetch = [&](int64_t i) BLK_INLINE {
    load_raw(row, (const NX*)p.x + i * p.ldx, rx);
    if (p.f) load_raw(row, (const NB*)p.f + i * p.ldf, rf);
    if (p.gate) load_raw(row, (const NB*)p.gate + (int64_t)((uint32_t)i / a.rows_per_gate) * p.ldgate, rg);
  };
  if (m < p.M) fetch(m);
  for (; m < p.M; m += step) {                           // (a row's lanes leave together; L > 64: the workgroup)
    float s[P], f[P], g[P];
    to_f32(rx, s);
    if (p.f) to_f32(rf, f);
    if (p.gate) to_f32(rg, g);
    if (m + step < p.M) fetch(m + step);
    if (p.f) {
      if (p.post != DPVO_NORM_NONE) {
        row.normalise(f, p.post, p.post_eps);
#pragma unroll
        for (int e = 0; e < P; ++e) f[e] = f[e] * pw[e] + pb[e];
      }
      if (p.gate) {
        act_n<sizeof(NB) == 4, false, P>(p.gate_activation, g);
#pragma unroll
        for (int e = 0; e < P; ++e) s[e] += p.scale * (g[e] * f[e]);
      } else {
#pragma unroll
        for (int e = 0; e < P; ++e) s[e] += p.scale * f[e];
      }
    }
    if (p.s) row.store((NX*)p.s + m * p.D, s);
    if (p.norm == DPVO_NORM_NONE) continue;
    row.normalise(s, p.norm, p.eps);
#pragma unroll
    for (int e = 0; e < P; ++e) s[e] = s[e] * w[e] + b[e];
    if (p.h_dtype == p.x_dtype) row.store((NX*)p.h + m * p.D, s);
    else row.store((NB*)p.h + m * p.D, s);
  }
}

// ---- sums over a workgroup's rows of what each lane finds for its columns.  In LDS where they fit (each thread its own 16-byte pieces, in an
// order that touches every bank once): five arrays of them in registers leave room for two waves on a SIMD only, and for spills.
template <int T, int P, bool IN_LDS> struct Sums {
  float reg[IN_LDS ? 1 : P];
  f4* lds;
  __device__ __forceinline__ void init(bool on, float*& room) {
    if constexpr (IN_LDS) {
      lds = on ? (f4*)room + threadIdx.x : nullptr;
      if (on) {
#pragma unroll
        for (int q = 0; q < P / 4; ++q) lds[q * T] = f4{0.f, 0.f, 0.f, 0.f};
        room += T * P;
      }
    } else {
#pragma unroll
      for (int e = 0; e < P; ++e) reg[e] = 0.f;
    }
  }
  __device__ __forceinline__ void add(bool on, const float (&v)[P]) {
    if constexpr (IN_LDS) {
      if (!on) return;
#pragma unroll
      for (int q = 0; q < P / 4; ++q) lds[q * T] += f4{v[q * 4], v[q * 4 + 1], v[q * 4 + 2], v[q * 4 + 3]};
    } else {
#pragma unroll
      for (int e = 0; e < P; ++e) reg[e] += v[e];
    }
  }
  // to `out` [D], and back to zero.  SLOTS > 1 (always in LDS): summed over the row slots, in order
  template <class R> __device__ __forceinline__ void flush(const R& row, float* out) {
    if constexpr (R::SLOTS == 1) {
      float v[P];
#pragma unroll
      for (int e = 0; e < P; ++e) {
        if constexpr (IN_LDS) v[e] = lds[e / 4 * T][e % 4];
        else v[e] = reg[e];
      }
      row.store(out, v);
      if constexpr (IN_LDS) {
#pragma unroll
        for (int q = 0; q < P / 4; ++q) lds[q * T] = f4{0.f, 0.f, 0.f, 0.f};
      } else {
#pragma unroll
        for (int e = 0; e < P; ++e) reg[e] = 0.f;
      }
    } else {
      constexpr int L = T / R::SLOTS;
      __syncthreads();
      const f4* all = lds - threadIdx.x;
      for (int i = threadIdx.x; i < L * P; i += T) {     // element i / L of lane i % L
        const int l = i % L, e = i / L, c = (l + e / R::PIECE * L) * R::PIECE + e % R::PIECE;
        if (c < row.D) {
          float v = 0.f;
#pragma unroll
          for (int k = 0; k < R::SLOTS; ++k) v += all[e / 4 * T + k * L + l][e % 4];
          out[c] = v;
        }
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < P / 4; ++q) lds[q * T] = f4{0.f, 0.f, 0.f, 0.f};
    }
  }
};

// 16-bit rows in pieces of 8: four waves to a SIMD at the price of some thirty spilled registers (8192 x 4096 with both norms: 113 us against
// 143 with the two that fit without; f32 streams spill more and lose: 138 against 99 us at 45312 x 384)
template <class NX, class NB, int L, int V, int E, bool IN_LDS> __global__ void __launch_bounds__(threads<L>(), sizeof(NX) == 2 && E == 8 ? 4 : 1) norm_back_kernel(const NormArgs a) {
  typedef Row<L, V, E, sizeof(NX) == 4> R;
  constexpr int P = R::P, T = threads<L>();
  __shared__ float red[4 * R::WPR];
  extern __shared__ __attribute__((aligned(16))) float sums[];
  const dpvo_residual_norm_t& p = a.p;
  R row(p.D, red);
  const bool norm = p.norm != DPVO_NORM_NONE && p.dh, post = p.f && p.post != DPVO_NORM_NONE;
  Sums<T, P, IN_LDS> aw, ab, apw, apb, ag;
  float* room = sums;
  aw.init(p.dw, room);
  ab.init(p.db, room);
  apw.init(p.dpw, room);
  apb.init(p.dpb, room);
  ag.init(a.part_gate, room);
  // the weights stay in registers where there is room
  constexpr bool KEEP = L < 1024;
  float kw[P], kpw[P];
  if constexpr (KEEP) {
    row.param(p.w, p.w_dtype, 1.f, kw);
    row.param(p.pw, p.w_dtype, 1.f, kpw);
  }
  const int64_t g0 = blockIdx.x / a.bpg * a.gpb, part = blockIdx.x % a.bpg;
  const int64_t g1 = g0 + a.gpb < a.groups ? g0 + a.gpb : a.groups;
  // this workgroup's rounds (SLOTS rows each) of each of its groups
  const int64_t rounds = (a.rpg + R::SLOTS - 1) / R::SLOTS, k0 = rounds * part / a.bpg, k1 = rounds * (part + 1) / a.bpg;
  Raw<NX, P> rx, rs, rhx;
  Raw<NB, P> rf, rg, rhb;                                // (rhx and rhb are one where the types are)
  constexpr bool ONE = __is_same(NX, NB);
  const bool hx = p.h_dtype == p.x_dtype;
  auto fetch = [&](int64_t g, int64_t k) BLK_INLINE {
    const int64_t in = k * R::SLOTS + row.slot, i = g * a.rpg + in;
    if (in >= a.rpg) return;
    load_raw(row, (const NX*)p.x + i * p.ldx, rx);
    if (p.f) load_raw(row, (const NB*)p.f + i * p.ldf, rf);
    if (p.gate) load_raw(row, (const NB*)p.gate + (a.shared ? g : i) * p.ldgate, rg);
    if (norm) {
      if (ONE || hx) load_raw(row, (const NX*)p.dh + i * p.lddh, rhx);
      else load_raw(row, (const NB*)p.dh + i * p.lddh, rhb);
    }
    if (p.ds) load_raw(row, (const NX*)p.ds + i * p.ldds, rs);
  };
  if (k0 < k1 && g0 < g1) fetch(g0, k0);
  for (int64_t g = g0; g < g1; ++g) {
    for (int64_t k = k0; k < k1; ++k) {
      const int64_t in = k * R::SLOTS + row.slot, m = g * a.rpg + in;
      float s[P], f[P], ga[P], gd[P], d[P], ds[P], t[P];
      to_f32(rx, s);
      if (p.f) to_f32(rf, f);
      if (p.gate) to_f32(rg, gd);
#pragma unroll
      for (int e = 0; e < P; ++e) d[e] = ds[e] = 0.f;
      if (norm) {
        if (ONE || hx) to_f32(rhx, d);
        else to_f32(rhb, d);
      }
      if (p.ds) to_f32(rs, ds);
      if (k + 1 < k1) fetch(g, k + 1);
      else if (g + 1 < g1) fetch(g + 1, k0);
      if (in >= a.rpg) continue;                         // (a row's lanes together; never with L > 64)

      float fr = 0.f;
      if (p.f) {
        if (post) {
          fr = row.normalise(f, p.post, p.post_eps);
          if constexpr (!KEEP) row.param(p.pw, p.w_dtype, 1.f, kpw);
          row.param(p.pb, p.w_dtype, 0.f, t);
#pragma unroll
          for (int e = 0; e < P; ++e) t[e] = f[e] * kpw[e] + t[e];
        } else {
#pragma unroll
          for (int e = 0; e < P; ++e) t[e] = f[e];
        }
        if (p.gate) {
          act_d_n<sizeof(NB) == 4, false, P>(p.gate_activation, gd, ga);
        } else {
#pragma unroll
          for (int e = 0; e < P; ++e) {
            ga[e] = 1.f;
            gd[e] = 0.f;
          }
        }
#pragma unroll
        for (int e = 0; e < P; ++e) {
          s[e] += p.scale * (ga[e] * t[e]);
          gd[e] *= t[e];
        }
      }
      if (norm) {
        const float r = row.normalise(s, p.norm, p.eps);
        if constexpr (!KEEP) row.param(p.w, p.w_dtype, 1.f, kw);
        ab.add(p.db, d);
#pragma unroll
        for (int e = 0; e < P; ++e) {
          t[e] = d[e] * s[e];
          d[e] *= kw[e];
        }
        aw.add(p.dw, t);
        row.back(d, s, r, p.norm);
      }
#pragma unroll
      for (int e = 0; e < P; ++e) d[e] += ds[e];
      if (p.dx) row.store((NX*)p.dx + m * p.D, d);
      if (!p.f) continue;
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const float q = p.scale * d[e];
        d[e] = q * ga[e];                                // gradient of post(f)
        gd[e] *= q;                                      // ... of the gate
      }
      if (a.part_gate) ag.add(true, gd);
      else if (p.dgate) row.store((NB*)p.dgate + m * p.D, gd);
      if (post) {
        if constexpr (!KEEP) row.param(p.pw, p.w_dtype, 1.f, kpw);
        apb.add(p.dpb, d);
#pragma unroll
        for (int e = 0; e < P; ++e) {
          t[e] = d[e] * f[e];
          d[e] *= kpw[e];
        }
        apw.add(p.dpw, t);
        if (p.df) row.back(d, f, fr, p.post);
      }
      if (p.df) row.store((NB*)p.df + m * p.D, d);
    }
    if (a.part_gate) ag.flush(row, a.part_gate + (g * a.bpg + part) * p.D);
  }
  const int64_t o = (int64_t)blockIdx.x * p.D;
  if (p.dw) aw.flush(row, a.part_w + o);
  if (p.db) ab.flush(row, a.part_b + o);
  if (p.dpw) apw.flush(row, a.part_pw + o);
  if (p.dpb) apb.flush(row, a.part_pb + o);
}

template <class NX, class NB, int I> int norm_go(const NormArgs& a, bool back, int64_t blocks, hipStream_t s) {
  constexpr NormShape S = NORM_SHAPES[I];
  constexpr int T = threads<S.L>();
  if (!back) {
    hipLaunchKernelGGL((norm_kernel<NX, NB, S.L, S.V, S.E>), dim3((unsigned)blocks), dim3(T), 0, s, a);
  } else {
    const dpvo_residual_norm_t& p = a.p;
    const int n = (p.dw != nullptr) + (p.db != nullptr) + (p.dpw != nullptr) + (p.dpb != nullptr) + (a.part_gate != nullptr);
    constexpr int one = T * S.V * S.E * 4;
    // 160 KB of LDS: five arrays always fit up to D = 4096, above that as many as are asked for may not
    if (n * one <= 160 * 1024 - 256) {
      auto k = norm_back_kernel<NX, NB, S.L, S.V, S.E, true>;
      if (n * one > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024 - 256);
        if (e != hipSuccess) return (int)e;
      }
      hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(T), n * one, s, a);
    } else if constexpr (5 * one > 160 * 1024 - 256) {
      hipLaunchKernelGGL((norm_back_kernel<NX, NB, S.L, S.V, S.E, false>), dim3((unsigned)blocks), dim3(T), 0, s, a);
    }
  }
  DPVO_LAUNCH_CHECK();
  return DPVO_OK;
}
template <class NX, class NB> int norm_pick(const NormArgs& a, int shape, bool back, int64_t blocks, hipStream_t s) {
  switch (shape) {
#define BLK_CASE(I) case I: return norm_go<NX, NB, I>(a, back, blocks, s);
    BLK_CASE(0) BLK_CASE(1) BLK_CASE(2) BLK_CASE(3) BLK_CASE(4) BLK_CASE(5) BLK_CASE(6) BLK_CASE(7) BLK_CASE(8) BLK_CASE(9)
    BLK_CASE(10) BLK_CASE(11)
#undef BLK_CASE
  }
  return DPVO_E_UNSUPPORTED;
}

}  // namespace
}  // namespace blk
