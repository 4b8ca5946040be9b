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
// Rows of up to 4096 elements: a row lives in the registers of L lanes, so every tensor is read once and statistics are two-pass in f32 at no traffic;
// the next row's loads are under way while a row is computed.  Nothing but memory bounds the forward kernels.  Gradients of what all rows (of a group)
// share are summed in LDS over a workgroup's rows, then over its row slots, then over workgroups by a second launch: no atomics, the order is
// fixed; the sums in LDS and spilled registers bound the backward.  Wider rows: what does
// not fit the registers is read again from L2, and backward the sums over rows are a second kernel, which reads the inputs again (below).
// Measured: 45312 x 384 with f32 stream, f16 branch and gate forward 46 us (5.3 TB/s; a large copy reaches 5.0 to 6.8); 8192 x 4096 bf16 with both
// norms and a gate for each of four groups forward 54 us (5.0 TB/s), backward 115 + 6 us (3.5 TB/s).
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
  float* stats;                                          // wide rows: NORM_STATS of each row, from the first backward kernel to the second
};
constexpr int NORM_STATS = 6;

int norm_f16(const NormArgs& a, int shape, bool back, int64_t blocks, hipStream_t st);     // branch types; stream: the same or f32
int norm_bf16(const NormArgs& a, int shape, bool back, int64_t blocks, hipStream_t st);
int norm_f32(const NormArgs& a, int shape, bool back, int64_t blocks, hipStream_t st);

namespace {

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

// A lane's elements as they are stored
template <class T, int P> struct Raw { T v[P]; };

// The lanes of a row: V pieces of 8 each.  RAGGED: the piece that the row's end would cut is the row's last 8 elements instead, of which the first
// ones belong to its neighbour and count as zeros.  (Guards on its elements' loads would make its wave, and at the next barrier the others, wait
// for each tensor in turn.)  Below 8 elements there is one lane, with guards.
template <int L, int V, bool RAGGED, bool FINE> struct Row {
  static constexpr int E = 8, P = V * E;                 // elements of a piece, of a lane
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
  __device__ __forceinline__ bool has(int i) const { return (lane + i * L) * E < D; }
  __device__ __forceinline__ int col(int i) const {
    const int c = (lane + i * L) * E;
    return RAGGED && c + E > D && D >= E ? D - E : c;
  }
  __device__ __forceinline__ int first(int i) const { return RAGGED ? (lane + i * L) * E - col(i) : 0; }     // own element of a piece that is there
  __device__ __forceinline__ bool in(int i, int e) const { return has(i) && (!RAGGED || (e >= first(i) && e < D)); }
  // piece i of a row at p: as it lies there; as f32, zeros where there is no own element; and to it
  template <class T> __device__ __forceinline__ void fetch(const T* p, int i, T* o) const {
    if (has(i) && (!RAGGED || D >= E)) {
      __builtin_memcpy(o, p + col(i), sizeof(T) * E);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = RAGGED && in(i, e) ? p[e] : (T)0.f;
    }
  }
  template <class T> __device__ __forceinline__ void own(const T* t, int i, float* o) const {
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = !RAGGED || in(i, e) ? (float)t[e] : 0.f;
  }
  template <class T> __device__ __forceinline__ void piece(const T* p, int i, float* o) const {
    T t[E];
    fetch(p, i, t);
    own(t, i, o);
  }
  template <class T> __device__ __forceinline__ void put(T* p, int i, const float* v) const {
    if (!has(i)) return;
    T t[E];
#pragma unroll
    for (int e = 0; e < E; ++e) t[e] = (T)v[e];
    if (!RAGGED || (first(i) == 0 && D >= E)) {
      __builtin_memcpy(p + col(i), t, sizeof(t));
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (in(i, e)) p[col(i) + e] = t[e];
    }
  }
  // of a parameter, `none` without one
  __device__ __forceinline__ void param(const void* p, int type, float none, int i, float* o) const {
    if (!p) {
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = none;
    }
    else if (type == DPVO_F32) piece((const float*)p, i, o);
    else if (type == DPVO_F16) piece((const _Float16*)p, i, o);
    else piece((const __bf16*)p, i, o);
  }
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
    for (int i = 0; i < V; ++i) put(p, i, v + i * E);
  }
  __device__ __forceinline__ void param(const void* p, int type, float none, float (&o)[P]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) param(p, type, none, i, o + i * E);
  }
  // v -> its normalised row (before weights); returns the row's factor, m: its mean (0: rms).  Elements behind D stay 0.
  __device__ __forceinline__ float normalise(float (&v)[P], int kind, float eps, float& m) {
    m = 0.f;
    if (kind == DPVO_NORM_LAYER) {
#pragma unroll
      for (int e = 0; e < P; ++e) m += v[e];
      m = sum(m) * inv;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float& x = v[i * E + e];
        x = in(i, e) ? x - m : 0.f;
        q += x * x;
      }
    q = sum(q) * inv + eps;
    const float r = FINE ? 1.f / sqrtf(q) : __builtin_amdgcn_rsqf(q);   // (rsq: one unit in the last place of f32)
#pragma unroll
    for (int e = 0; e < P; ++e) v[e] *= r;
    return r;
  }
  __device__ __forceinline__ float normalise(float (&v)[P], int kind, float eps) {
    float m;
    return normalise(v, kind, eps, m);
  }
  // d (gradient behind the weights, 0 behind D) -> gradient of the row; xh: the normalised row; a, b: the two means
  __device__ __forceinline__ void back(float (&d)[P], const float (&xh)[P], float r, int kind, float& a, float& b) {
    a = b = 0.f;
#pragma unroll
    for (int e = 0; e < P; ++e) {
      a += d[e];
      b += d[e] * xh[e];
    }
    sum(a, b);
    a = kind == DPVO_NORM_LAYER ? a * inv : 0.f;
    b *= inv;
#pragma unroll
    for (int i = 0; i < V; ++i)                          // (behind D the mean alone would be left, and reach the next sum)
#pragma unroll
      for (int e = 0; e < E; ++e) d[i * E + e] = in(i, e) ? r * (d[i * E + e] - a - xh[i * E + e] * b) : 0.f;
  }
  __device__ __forceinline__ void back(float (&d)[P], const float (&xh)[P], float r, int kind) {
    float a, b;
    back(d, xh, r, kind, a, b);
  }
};

template <class T, class R> __device__ __forceinline__ void load_raw(const R& row, const T* p, Raw<T, R::P>& o) {
#pragma unroll
  for (int i = 0; i < R::P / R::E; ++i) row.fetch(p, i, o.v + i * R::E);
}
template <class T, class R> __device__ __forceinline__ void to_f32(const R& row, const Raw<T, R::P>& r, float (&o)[R::P]) {
#pragma unroll
  for (int i = 0; i < R::P / R::E; ++i) row.own(r.v + i * R::E, i, o + i * R::E);
}

template <class NX, class NB, int L, bool RAGGED> __global__ void __launch_bounds__(threads<L>()) norm_kernel(const NormArgs a) {
  typedef Row<L, 1, RAGGED, sizeof(NX) == 4> R;
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
    to_f32(row, rx, s);
    if (p.f) to_f32(row, rf, f);
    if (p.gate) to_f32(row, rg, g);
    if (m + step < p.M) fetch(m + step);
    if (p.f) {
      if (p.post != DPVO_NORM_NONE) {
        row.normalise(f, p.post, p.post_eps);
#pragma unroll
        for (int e = 0; e < P; ++e) f[e] = f[e] * pw[e] + pb[e];
      }
      if (p.gate) {
        act_n<sizeof(NX) == 4, false, P>(p.gate_activation, g);
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

// ---- sums over a workgroup's rows of what each lane finds for its columns, in LDS (each thread its own 16-byte pieces, in an order that
// touches every bank once): five arrays of them in registers would leave room for two waves on a SIMD only, and for spills.
template <int T, int P> struct Sums {
  f4* lds;
  __device__ __forceinline__ void init(bool on, float*& room) {
    lds = on ? (f4*)room + threadIdx.x : nullptr;
    if (on) {
      clear();
      room += T * P;
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int q = 0; q < P / 4; ++q) lds[q * T] = f4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void add(bool on, const float (&v)[P]) {
    if (!on) return;
#pragma unroll
    for (int q = 0; q < P / 4; ++q) lds[q * T] += f4{v[q * 4], v[q * 4 + 1], v[q * 4 + 2], v[q * 4 + 3]};
  }
  // to `out` [D], and back to zero; SLOTS > 1: summed over the row slots, in order
  template <class R> __device__ __forceinline__ void flush(const R& row, float* out) {
    if constexpr (R::SLOTS == 1) {
      float v[P];
#pragma unroll
      for (int e = 0; e < P; ++e) v[e] = lds[e / 4 * T][e % 4];
      row.store(out, v);
    } else {
      constexpr int L = T / R::SLOTS;
      __syncthreads();
      const f4* all = lds - threadIdx.x;
      for (int i = threadIdx.x; i < L * P; i += T) {     // element i / L of lane i % L
        const int l = i % L, e = i / L, c0 = l * R::E;
        const int c = (c0 + R::E > row.D && row.D >= R::E ? row.D - R::E : c0) + e;   // (as Row::col)
        if (c0 <= c && c < row.D) {
          float v = 0.f;
#pragma unroll
          for (int k = 0; k < R::SLOTS; ++k) v += all[e / 4 * T + k * L + l][e % 4];
          out[c] = v;
        }
      }
      __syncthreads();
    }
    clear();
  }
};

// 16-bit rows: four waves to a SIMD at the price of some thirty spilled registers (8192 x 4096 with both norms: 113 us against 143 with the
// two that fit without; f32 streams spill more and lose: 138 against 99 us at 45312 x 384, and so do ragged rows: 223 against 135 at 4096 x 2333)
template <class NX, class NB, int L, bool RAGGED> __global__ void __launch_bounds__(threads<L>(), sizeof(NX) == 2 && !RAGGED ? 4 : 1) norm_back_kernel(const NormArgs a) {
  typedef Row<L, 1, RAGGED, sizeof(NX) == 4> R;
  constexpr int P = R::P, T = threads<L>();
  __shared__ float red[4 * R::WPR];
  extern __shared__ __attribute__((aligned(16))) float sums[];
  const dpvo_residual_norm_t& p = a.p;
  R row(p.D, red);
  const bool norm = p.norm != DPVO_NORM_NONE && p.dh, post = p.f && p.post != DPVO_NORM_NONE;
  Sums<T, P> aw, ab, apw, apb, ag;
  float* room = sums;
  aw.init(p.dw, room);
  ab.init(p.db, room);
  apw.init(p.dpw, room);
  apb.init(p.dpb, room);
  ag.init(a.part_gate, room);
  // The weights stay in registers up to 512 lanes: 8192 x 4096 bf16 104 us, read again for each row 117; 45312 x 384 64 and 72, f32 97 and 119; narrow
  // rows of 16 bits lose (131072 x 128: 92 and 59), and 1024 lanes would gain (4096 x 8192 bf16 121 us kept, 131 read again).
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
      to_f32(row, rx, s);
      if (p.f) to_f32(row, rf, f);
      if (p.gate) to_f32(row, rg, gd);
#pragma unroll
      for (int e = 0; e < P; ++e) d[e] = ds[e] = 0.f;
      if (norm) {
        if (ONE || hx) to_f32(row, rhx, d);
        else to_f32(row, rhb, d);
      }
      if (p.ds) to_f32(row, rs, ds);
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
          act_d_n<sizeof(NX) == 4, false, P>(p.gate_activation, gd, ga);
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

// piece i of a branch behind its norm's weights
template <class R> __device__ __forceinline__ void wide_post(const R& row, const dpvo_residual_norm_t& p, int i, const float* f, float (&o)[R::E]) {
  if (p.post == DPVO_NORM_NONE) {
#pragma unroll
    for (int e = 0; e < R::E; ++e) o[e] = f[e];
  } else {
    float t[R::E];
    row.param(p.pw, p.w_dtype, 1.f, i, o);
    row.param(p.pb, p.w_dtype, 0.f, i, t);
#pragma unroll
    for (int e = 0; e < R::E; ++e) o[e] = f[e] * o[e] + t[e];
  }
}
// ---- rows of more than 4096 elements: a workgroup of 1024 threads to a row, V pieces of 8 on each.  Only the normalised rows and the gradient stay
// in registers (16 elements of everything that a row needs would not fit); what is needed again is read again, from L2.
template <class NX, class NB, int L, int V, bool RAGGED> __global__ void __launch_bounds__(L, 4) norm_wide_kernel(const NormArgs a) {
  typedef Row<L, V, RAGGED, sizeof(NX) == 4> R;
  constexpr int P = R::P, E = R::E;
  __shared__ float red[4 * R::WPR];
  const dpvo_residual_norm_t& p = a.p;
  R row(p.D, red);
  for (int64_t m = blockIdx.x; m < p.M; m += gridDim.x) {
    float s[P], f[P];
    Raw<NX, P> rx;
    load_raw(row, (const NX*)p.x + m * p.ldx, rx);
    if (p.f) {
      Raw<NB, P> rf;
      load_raw(row, (const NB*)p.f + m * p.ldf, rf);
      to_f32(row, rf, f);
      if (p.post != DPVO_NORM_NONE) row.normalise(f, p.post, p.post_eps);
    }
    to_f32(row, rx, s);
    if (p.f) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (!row.has(i)) continue;
          float t[E], u[E];
        wide_post(row, p, i, f + i * E, t);
        if (p.gate) {
          row.piece((const NB*)p.gate + (int64_t)((uint32_t)m / a.rows_per_gate) * p.ldgate, i, u);
          act_n<sizeof(NX) == 4, false, E>(p.gate_activation, u);
#pragma unroll
          for (int e = 0; e < E; ++e) t[e] *= u[e];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) s[i * E + e] += p.scale * t[e];
      }
    }
    if (p.s) row.store((NX*)p.s + m * p.D, s);
    if (p.norm == DPVO_NORM_NONE) continue;
    row.normalise(s, p.norm, p.eps);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (!row.has(i)) continue;
      float t[E], u[E];
      row.param(p.w, p.w_dtype, 1.f, i, t);
      row.param(p.b, p.w_dtype, 0.f, i, u);
#pragma unroll
      for (int e = 0; e < E; ++e) t[e] = s[i * E + e] * t[e] + u[e];
      if (p.h_dtype == p.x_dtype) row.put((NX*)p.h + m * p.D, i, t);
      else row.put((NB*)p.h + m * p.D, i, t);
    }
  }
}

// backward, first kernel: dx, df and a gate gradient of its own for each row; the rows' statistics for the second
template <class NX, class NB, int L, int V, bool RAGGED> __global__ void __launch_bounds__(L, 4) norm_wide_back_kernel(const NormArgs a) {
  typedef Row<L, V, RAGGED, sizeof(NX) == 4> R;
  constexpr int P = R::P, E = R::E;
  __shared__ float red[4 * R::WPR];
  const dpvo_residual_norm_t& p = a.p;
  R row(p.D, red);
  const bool norm = p.norm != DPVO_NORM_NONE && p.dh, post = p.f && p.post != DPVO_NORM_NONE, hx = p.h_dtype == p.x_dtype;
  for (int64_t m = blockIdx.x; m < p.M; m += gridDim.x) {
    float s[P], f[P], d[P];
    float ms = 0.f, rs = 0.f, av = 0.f, bv = 0.f, mf = 0.f, rf = 0.f;
    const NB* gate = p.gate ? (const NB*)p.gate + (a.shared ? m / a.rpg : m) * p.ldgate : nullptr;
    if (p.f) {
      Raw<NB, P> r;
      load_raw(row, (const NB*)p.f + m * p.ldf, r);
      to_f32(row, r, f);
      if (post) rf = row.normalise(f, p.post, p.post_eps, mf);
    }
#pragma unroll
    for (int e = 0; e < P; ++e) d[e] = 0.f;
    if (norm) {
      Raw<NX, P> r;
      load_raw(row, (const NX*)p.x + m * p.ldx, r);
      to_f32(row, r, s);
      if (p.f) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (!row.has(i)) continue;
              float t[E], u[E];
          wide_post(row, p, i, f + i * E, t);
          if (gate) {
            row.piece(gate, i, u);
            act_n<sizeof(NX) == 4, false, E>(p.gate_activation, u);
#pragma unroll
            for (int e = 0; e < E; ++e) t[e] *= u[e];
          }
#pragma unroll
          for (int e = 0; e < E; ++e) s[i * E + e] += p.scale * t[e];
        }
      }
      rs = row.normalise(s, p.norm, p.eps, ms);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (!row.has(i)) continue;
          float t[E], u[E];
        if (hx) row.piece((const NX*)p.dh + m * p.lddh, i, t);
        else row.piece((const NB*)p.dh + m * p.lddh, i, t);
        row.param(p.w, p.w_dtype, 1.f, i, u);
#pragma unroll
        for (int e = 0; e < E; ++e) d[i * E + e] = t[e] * u[e];
      }
      row.back(d, s, rs, p.norm, av, bv);
    }
    if (a.stats && threadIdx.x == 0) {
      float* o = a.stats + m * NORM_STATS;
      o[0] = ms, o[1] = rs, o[2] = av, o[3] = bv, o[4] = mf, o[5] = rf;
    }
    if (p.ds) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (!row.has(i)) continue;
        float t[E];
        row.piece((const NX*)p.ds + m * p.ldds, i, t);
#pragma unroll
        for (int e = 0; e < E; ++e) d[i * E + e] += t[e];
      }
    }
    if (p.dx) row.store((NX*)p.dx + m * p.D, d);
    if (!p.df && !p.dgate) continue;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (!row.has(i)) continue;
      float* q = d + i * E;
#pragma unroll
      for (int e = 0; e < E; ++e) q[e] *= p.scale;
      if (gate) {
        float t[E], u[E], y[E];
        row.piece(gate, i, u);
        act_d_n<sizeof(NX) == 4, false, E>(p.gate_activation, u, y);
        if (p.dgate && !a.part_gate) {
          wide_post(row, p, i, f + i * E, t);
#pragma unroll
          for (int e = 0; e < E; ++e) t[e] *= q[e] * u[e];
          row.put((NB*)p.dgate + m * p.D, i, t);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) q[e] *= y[e];
      }
      if (post) {
        float t[E];
        row.param(p.pw, p.w_dtype, 1.f, i, t);
#pragma unroll
        for (int e = 0; e < E; ++e) q[e] *= t[e];
      }
    }
    if (!p.df) continue;
    if (post) row.back(d, f, rf, p.post);
    row.store((NB*)p.df + m * p.D, d);
  }
}

// ... second kernel: with the statistics every gradient that rows share is a sum over rows of a product of elements.  A thread has 8 columns (of
// 2048 in a workgroup), a workgroup the rows that norm_back_kernel gives one; the sums stay in registers.
template <class NX, class NB> __global__ void __launch_bounds__(256, 2) norm_cols_kernel(const NormArgs a) {
  typedef Row<256, 1, true, sizeof(NX) == 4> R;
  constexpr int E = R::E;
  const dpvo_residual_norm_t& p = a.p;
  R row(p.D, nullptr);
  row.lane += blockIdx.x * 256;                          // (of the row's piece of 2048)
  if (!row.has(0)) return;
  const bool norm = p.norm != DPVO_NORM_NONE && p.dh, post = p.f && p.post != DPVO_NORM_NONE, hx = p.h_dtype == p.x_dtype;
  const bool branch = a.part_gate || p.dpw || p.dpb;
  float w[E], pw[E], pb[E], aw[E] = {}, ab[E] = {}, apw[E] = {}, apb[E] = {}, ag[E] = {};
  row.param(p.w, p.w_dtype, 1.f, 0, w);
  row.param(p.pw, p.w_dtype, 1.f, 0, pw);
  row.param(p.pb, p.w_dtype, 0.f, 0, pb);
  const int64_t g0 = blockIdx.y / a.bpg * a.gpb, part = blockIdx.y % a.bpg;
  const int64_t g1 = g0 + a.gpb < a.groups ? g0 + a.gpb : a.groups;
  const int64_t k0 = a.rpg * part / a.bpg, k1 = a.rpg * (part + 1) / a.bpg;
  Raw<NX, E> rx, rs, rhx;                                // the next row
  Raw<NB, E> rf, rg, rhb;
  constexpr bool ONE = __is_same(NX, NB);
  float st[NORM_STATS];
  auto fetch = [&](int64_t g, int64_t k) BLK_INLINE {
    const int64_t m = g * a.rpg + k;
    load_raw(row, (const NX*)p.x + m * p.ldx, rx);
    if (p.f) load_raw(row, (const NB*)p.f + m * p.ldf, rf);
    if (p.gate) load_raw(row, (const NB*)p.gate + (a.shared ? g : m) * p.ldgate, rg);
    if (norm) {
      if (ONE || hx) load_raw(row, (const NX*)p.dh + m * p.lddh, rhx);
      else load_raw(row, (const NB*)p.dh + m * p.lddh, rhb);
    }
    if (branch && p.ds) load_raw(row, (const NX*)p.ds + m * p.ldds, rs);
#pragma unroll
    for (int i = 0; i < NORM_STATS; ++i) st[i] = a.stats[m * NORM_STATS + i];
  };
  if (k0 < k1 && g0 < g1) fetch(g0, k0);
  for (int64_t g = g0; g < g1; ++g) {
    for (int64_t k = k0; k < k1; ++k) {
      const float ms = st[0], r = st[1], av = st[2], bv = st[3], mf = st[4], fr = st[5];
      float s[E], f[E], t[E], ga[E], gd[E], d[E] = {}, q[E] = {};
      to_f32(row, rx, s);
      if (p.f) to_f32(row, rf, f);
      if (p.gate) to_f32(row, rg, gd);
      if (norm) {
        if (ONE || hx) to_f32(row, rhx, d);
        else to_f32(row, rhb, d);
      }
      if (branch && p.ds) to_f32(row, rs, q);
      if (k + 1 < k1) fetch(g, k + 1);
      else if (g + 1 < g1) fetch(g + 1, k0);
      if (p.f) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (post) f[e] = (f[e] - mf) * fr;
          t[e] = post ? f[e] * pw[e] + pb[e] : f[e];
        }
        if (p.gate) {
          act_d_n<sizeof(NX) == 4, false, E>(p.gate_activation, gd, ga);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) ga[e] = 1.f, gd[e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] += p.scale * (ga[e] * t[e]);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (!norm) break;
        const float xh = (s[e] - ms) * r;
        ab[e] += d[e];
        aw[e] += d[e] * xh;
        q[e] += r * (d[e] * w[e] - av - xh * bv);
      }
      if (branch) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          q[e] *= p.scale;
          ag[e] += q[e] * (gd[e] * t[e]);
          q[e] *= ga[e];
          apb[e] += q[e];
          apw[e] += q[e] * f[e];
        }
      }
    }
    if (a.part_gate) {
      row.put(a.part_gate + (g * a.bpg + part) * p.D, 0, ag);
#pragma unroll
      for (int e = 0; e < E; ++e) ag[e] = 0.f;
    }
  }
  const int64_t o = (int64_t)blockIdx.y * p.D;
  if (p.dw) row.put(a.part_w + o, 0, aw);
  if (p.db) row.put(a.part_b + o, 0, ab);
  if (p.dpw) row.put(a.part_pw + o, 0, apw);
  if (p.dpb) row.put(a.part_pb + o, 0, apb);
}

// (512 threads with 16 elements each where those are enough, as two workgroups on a compute unit take turns at their barriers; 1024 with 16 for wider
// rows.  Whole pieces, bf16, forward and first backward kernel: 4096 x 8192 75 and 126 us, 2048 x 16384 73 and 143)
template <class NX, class NB, int L, bool RAGGED> int norm_wide(const NormArgs& a, bool back, int64_t blocks, hipStream_t s) {
  const dim3 rows((unsigned)(a.p.M < 8192 ? a.p.M : 8192));
  if (!back) hipLaunchKernelGGL((norm_wide_kernel<NX, NB, L, 2, RAGGED>), rows, dim3(L), 0, s, a);
  else hipLaunchKernelGGL((norm_wide_back_kernel<NX, NB, L, 2, RAGGED>), rows, dim3(L), 0, s, a);
  if (back && a.stats) hipLaunchKernelGGL((norm_cols_kernel<NX, NB>), dim3((unsigned)cdiv64(a.p.D, 2048), (unsigned)blocks), dim3(256), 0, s, a);
  DPVO_LAUNCH_CHECK();
  return DPVO_OK;
}
template <class NX, class NB, int I> int norm_go(const NormArgs& a, bool back, int64_t blocks, hipStream_t s) {
  constexpr NormShape S = NORM_SHAPES[I];
  constexpr int T = threads<S.L>();
  if (!back) {
    if constexpr (S.L < 1024) hipLaunchKernelGGL((norm_kernel<NX, NB, S.L, S.ragged>), dim3((unsigned)blocks), dim3(T), 0, s, a);
  } else {
    auto k = norm_back_kernel<NX, NB, S.L, S.ragged>;
    constexpr int one = T * 8 * 4, most = (S.L < 1024 ? 5 : 4) * one;   // 80 or 128 KB
    const int bytes = norm_sums(a.p, a.shared) * one;
    if (bytes > 64 * 1024) {                             // (always the same value: another thread may be about to launch)
      const hipError_t e = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, most);
      if (e != hipSuccess) return (int)e;
    }
    hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(T), bytes, s, a);
  }
  DPVO_LAUNCH_CHECK();
  return DPVO_OK;
}
template <class NX, class NB> int norm_pick(const NormArgs& a, int shape, bool back, int64_t blocks, hipStream_t s) {
  switch (shape) {
#define BLK_CASE(I) case I: return norm_go<NX, NB, I>(a, back, blocks, s);
    BLK_CASE(0) BLK_CASE(1) BLK_CASE(2) BLK_CASE(3) BLK_CASE(4) BLK_CASE(5) BLK_CASE(6) BLK_CASE(7) BLK_CASE(8) BLK_CASE(9) BLK_CASE(10) BLK_CASE(11)
#undef BLK_CASE
    case NORM_1024:
      if constexpr (sizeof(NX) == 2) return norm_go<NX, NB, NORM_1024>(a, back, blocks, s);
  }
  if (a.p.D % 8) return a.p.D <= 8192 ? norm_wide<NX, NB, 512, true>(a, back, blocks, s) : norm_wide<NX, NB, 1024, true>(a, back, blocks, s);
  return a.p.D <= 8192 ? norm_wide<NX, NB, 512, false>(a, back, blocks, s) : norm_wide<NX, NB, 1024, false>(a, back, blocks, s);
}

}  // namespace
}  // namespace blk
