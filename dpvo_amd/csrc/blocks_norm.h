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
// A row lives in the registers of L lanes, V pieces of 8 elements each, so every tensor is read once and statistics are two-pass in f32 at no
// traffic.  Nothing but memory bounds these kernels.  Gradients of what all rows (of a group) share are summed in registers over a workgroup's
// rows, then over its row slots through LDS, then over workgroups by a second launch: no atomics, the order is fixed.
#pragma once
#include "blocks_dev.h"

namespace blk {

struct NormArgs {
  dpvo_residual_norm_t p;
  int64_t rows_per_gate;                                 // rows that share a gate row
  // backward: a workgroup makes `gpb` whole groups of `rpg` rows, or (bpg > 1) one of the bpg parts of one group
  int64_t groups, rpg, gpb, bpg;
  float *part_gate, *part_w, *part_b, *part_pw, *part_pb;   // partial sums, a row of D each
};

// How a row of D elements is spread: V pieces of 8 on each of L lanes.  Few lanes for short rows (several rows a wave, short reductions),
// a workgroup for long ones.
struct NormShape { int L, V; };
inline NormShape norm_shape(int D) {
  if (D <= 128) return {16, 1};
  if (D <= 384) return {16, 3};
  if (D <= 512) return {64, 1};
  if (D <= 1024) return {64, 2};
  if (D <= 2048) return {64, 4};
  if (D <= 4096) return {256, 2};
  if (D <= 8192) return {256, 4};
  return {512, 4};
}
constexpr int NORM_MAX_D = 16384;
inline int norm_slots(const NormShape& s) { return s.L > 256 ? 1 : 256 / s.L; }

int norm_f16(const NormArgs& a, const NormShape& s, bool back, int64_t blocks, hipStream_t st);     // branch types; stream: the same or f32
int norm_bf16(const NormArgs& a, const NormShape& s, bool back, int64_t blocks, hipStream_t st);
int norm_f32(const NormArgs& a, const NormShape& s, bool back, int64_t blocks, hipStream_t st);

namespace {

__device__ __forceinline__ void param8(const void* p, int type, int64_t i, int nv, float (&o)[8]) {
  if (type == DPVO_F32) load_n<float, 8>((const float*)p + i, nv, o);
  else if (type == DPVO_F16) load_n<_Float16, 8>((const _Float16*)p + i, nv, o);
  else load_n<__bf16, 8>((const __bf16*)p + i, nv, o);
}

// sum over the L lanes that share a row; `red`: one float per wave of the workgroup (L > 64), used alternately
template <int L> __device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = (L < 64 ? L : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (L > 64) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[w] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < L / 64; ++i) v += red[i];
  }
  return v;
}

template <int L> constexpr int threads() { return L > 256 ? L : 256; }

template <class NX, class NB, int L, int V> struct Row {
  static constexpr int SLOTS = threads<L>() / L;         // rows at a time in a workgroup
  int lane, slot, D;
  float* red;                                            // [2][8] scratch for sums over waves
  int flip = 0;
  float inv;                                             // 1 / D

  __device__ __forceinline__ Row(int D_, float* red_) : lane(threadIdx.x % L), slot(threadIdx.x / L), D(D_), red(red_), inv(1.f / (float)D_) {}
  __device__ __forceinline__ int col(int i) const { return (lane + i * L) * 8; }
  __device__ __forceinline__ int nv(int i) const { const int n = D - col(i); return n < 0 ? 0 : n < 8 ? n : 8; }
  // consecutive sums use the two halves of the scratch in turn, so one barrier each is enough
  __device__ __forceinline__ float sum(float v) {
    flip ^= 8;
    return row_sum<L>(v, red + flip);
  }
  template <class T> __device__ __forceinline__ void load(const T* p, float (&o)[V][8]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) load_n<T, 8>(p + col(i), nv(i), o[i]);
  }
  template <class T> __device__ __forceinline__ void store(T* p, const float (&v)[V][8]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) store_n<T, 8>(p + col(i), nv(i), v[i]);
  }
  // v -> its normalised row (before weights); returns the row's factor.  Elements behind D stay 0.
  __device__ __forceinline__ float normalise(float (&v)[V][8], int kind, float eps) {
    float m = 0.f;
    if (kind == DPVO_NORM_LAYER) {
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) m += v[i][e];
      m = sum(m) * inv;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int n = nv(i);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[i][e] = e < n ? v[i][e] - m : 0.f;
        q += v[i][e] * v[i][e];
      }
    }
    const float r = 1.f / sqrtf(sum(q) * inv + eps);
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] *= r;
    return r;
  }
  // d (gradient behind the weights, 0 behind D) -> gradient of the row; xh: the normalised row
  __device__ __forceinline__ void back(float (&d)[V][8], const float (&xh)[V][8], float r, int kind) {
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        a += d[i][e];
        b += d[i][e] * xh[i][e];
      }
    a = kind == DPVO_NORM_LAYER ? sum(a) * inv : 0.f;
    b = sum(b) * inv;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) d[i][e] = r * (d[i][e] - a - xh[i][e] * b);
  }
};

// o = xh * w + b
template <int V, class R> __device__ __forceinline__ void affine(const R& R_, const void* w, const void* b, int type, const float (&xh)[V][8], float (&o)[V][8]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float t[8];
    const int n = R_.nv(i);
    if (w) {
      param8(w, type, R_.col(i), n, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[i][e] = xh[i][e] * t[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) o[i][e] = xh[i][e];
    }
    if (b) {
      param8(b, type, R_.col(i), n, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[i][e] += t[e];
    }
  }
}

template <class NX, class NB, int L, int V> __global__ void __launch_bounds__(threads<L>()) norm_kernel(const NormArgs a) {
  __shared__ float red[16];
  const dpvo_residual_norm_t& p = a.p;
  typedef Row<NX, NB, L, V> R;
  R row(p.D, red);
  for (int64_t m0 = (int64_t)blockIdx.x * R::SLOTS; m0 < p.M; m0 += (int64_t)gridDim.x * R::SLOTS) {
    const int64_t m = m0 + row.slot;
    if (L <= 64 && m >= p.M) return;                     // (whole lane groups leave; L > 64: one slot, never taken)
    float s[V][8];
    row.load((const NX*)p.x + m * p.ldx, s);
    if (p.f) {
      float f[V][8], g[V][8];
      row.load((const NB*)p.f + m * p.ldf, f);
      if (p.gate) row.load((const NB*)p.gate + m / a.rows_per_gate * p.ldgate, g);
      if (p.post != DPVO_NORM_NONE) {
        row.normalise(f, p.post, p.post_eps);
        affine<V>(row, p.pw, p.pb, p.w_dtype, f, f);
      }
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          s[i][e] += p.scale * (p.gate ? act_<sizeof(NB) == 4>(p.gate_activation, g[i][e]) * f[i][e] : f[i][e]);
    }
    if (p.s) row.store((NX*)p.s + m * p.D, s);
    if (p.norm == DPVO_NORM_NONE) continue;
    row.normalise(s, p.norm, p.eps);
    affine<V>(row, p.w, p.b, p.w_dtype, s, s);
    if (p.h_dtype == p.x_dtype) row.store((NX*)p.h + m * p.D, s);
    else row.store((NB*)p.h + m * p.D, s);
  }
}

// the workgroup's sum of a per-lane row of sums over its row slots, to `out` [D]
template <int L, int V, class R> __device__ __forceinline__ void flush(const R& row, float (&acc)[V][8], float* lds, float* out) {
  if constexpr (R::SLOTS == 1) {
    row.store(out, acc);
  } else {
    constexpr int W = L * V * 8;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < 8; e += 4) *(f4*)(lds + row.slot * W + row.col(i) + e) = f4{acc[i][e], acc[i][e + 1], acc[i][e + 2], acc[i][e + 3]};
    __syncthreads();
    for (int c = threadIdx.x; c < row.D; c += threads<L>()) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < R::SLOTS; ++k) v += lds[k * W + c];
      out[c] = v;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[i][e] = 0.f;
}

template <class NX, class NB, int L, int V> __global__ void __launch_bounds__(threads<L>()) norm_back_kernel(const NormArgs a) {
  __shared__ float red[16];
  typedef Row<NX, NB, L, V> R;
  __shared__ __attribute__((aligned(16))) float lds[R::SLOTS == 1 ? 4 : R::SLOTS * L * V * 8];
  const dpvo_residual_norm_t& p = a.p;
  R row(p.D, red);
  const bool layer = p.norm != DPVO_NORM_NONE, post = p.f && p.post != DPVO_NORM_NONE;
  float aw[V][8] = {}, ab[V][8] = {}, apw[V][8] = {}, apb[V][8] = {}, ag[V][8] = {};
  const int64_t g0 = blockIdx.x / a.bpg * a.gpb, part = blockIdx.x % a.bpg;
  const int64_t g1 = g0 + a.gpb < a.groups ? g0 + a.gpb : a.groups;
  for (int64_t g = g0; g < g1; ++g) {
    // this workgroup's rows of the group, whole rounds of SLOTS rows
    const int64_t rounds = (a.rpg + R::SLOTS - 1) / R::SLOTS, k0 = rounds * part / a.bpg, k1 = rounds * (part + 1) / a.bpg;
    for (int64_t k = k0; k < k1; ++k) {
      const int64_t in = k * R::SLOTS + row.slot;
      const int64_t m = g * a.rpg + in;
      if (in >= a.rpg || m >= p.M) continue;             // (whole lane groups; never with L > 64)
      float s[V][8], f[V][8], ga[V][8], gd[V][8], d[V][8];
      row.load((const NX*)p.x + m * p.ldx, s);
      float fr = 0.f;
      if (p.f) {
        row.load((const NB*)p.f + m * p.ldf, f);
        if (p.gate) row.load((const NB*)p.gate + m / a.rows_per_gate * p.ldgate, ga);
      }
      if (layer && p.dh) {
        if (p.h_dtype == p.x_dtype) row.load((const NX*)p.dh + m * p.lddh, d);
        else row.load((const NB*)p.dh + m * p.lddh, d);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) d[i][e] = 0.f;
      }
      if (p.f) {
        if (post) fr = row.normalise(f, p.post, p.post_eps);
        float pf[V][8];
        if (post) affine<V>(row, p.pw, p.pb, p.w_dtype, f, pf);
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float q = post ? pf[i][e] : f[i][e];
            if (p.gate) {
              const ActD t = act_d<sizeof(NB) == 4>(p.gate_activation, ga[i][e]);
              s[i][e] += p.scale * (t.y * q);
              ga[i][e] = t.y;
              gd[i][e] = t.d * q;
            } else {
              s[i][e] += p.scale * q;
              ga[i][e] = 1.f;
              gd[i][e] = 0.f;
            }
          }
      }
      if (layer && p.dh) {
        const float r = row.normalise(s, p.norm, p.eps);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float w[8];
          if (p.w) param8(p.w, p.w_dtype, row.col(i), row.nv(i), w);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (p.dw) aw[i][e] += d[i][e] * s[i][e];
            if (p.db) ab[i][e] += d[i][e];
            if (p.w) d[i][e] *= w[e];
          }
        }
        row.back(d, s, r, p.norm);
      }
      if (p.ds) {
        row.load((const NX*)p.ds + m * p.ldds, s);
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) d[i][e] += s[i][e];
      }
      if (p.dx) row.store((NX*)p.dx + m * p.D, d);
      if (!p.f) continue;
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float q = p.scale * d[i][e];
          d[i][e] = q * ga[i][e];                        // gradient of post(f)
          gd[i][e] *= q;                                 // ... of the gate
        }
      if (p.dgate) {
        if (a.part_gate) {
#pragma unroll
          for (int i = 0; i < V; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) ag[i][e] += gd[i][e];
        } else {
          row.store((NB*)p.dgate + m * p.D, gd);
        }
      }
      if (post) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float w[8];
          if (p.pw) param8(p.pw, p.w_dtype, row.col(i), row.nv(i), w);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (p.dpw) apw[i][e] += d[i][e] * f[i][e];
            if (p.dpb) apb[i][e] += d[i][e];
            if (p.pw) d[i][e] *= w[e];
          }
        }
        if (p.df) row.back(d, f, fr, p.post);
      }
      if (p.df) row.store((NB*)p.df + m * p.D, d);
    }
    if (a.part_gate) flush<L, V>(row, ag, lds, a.part_gate + (g * a.bpg + part) * p.D);
  }
  const int64_t o = (int64_t)blockIdx.x * p.D;
  if (p.dw) flush<L, V>(row, aw, lds, a.part_w + o);
  if (p.db) flush<L, V>(row, ab, lds, a.part_b + o);
  if (p.dpw) flush<L, V>(row, apw, lds, a.part_pw + o);
  if (p.dpb) flush<L, V>(row, apb, lds, a.part_pb + o);
}

template <class NX, class NB, int L, int V> int norm_go(const NormArgs& a, bool back, int64_t blocks, hipStream_t s) {
  if (back) hipLaunchKernelGGL((norm_back_kernel<NX, NB, L, V>), dim3((unsigned)blocks), dim3(threads<L>()), 0, s, a);
  else hipLaunchKernelGGL((norm_kernel<NX, NB, L, V>), dim3((unsigned)blocks), dim3(threads<L>()), 0, s, a);
  DPVO_LAUNCH_CHECK();
  return DPVO_OK;
}
template <class NX, class NB> int norm_pick(const NormArgs& a, const NormShape& sh, bool back, int64_t blocks, hipStream_t s) {
  switch (sh.L * 16 + sh.V) {
    case 16 * 16 + 1: return norm_go<NX, NB, 16, 1>(a, back, blocks, s);
    case 16 * 16 + 3: return norm_go<NX, NB, 16, 3>(a, back, blocks, s);
    case 64 * 16 + 1: return norm_go<NX, NB, 64, 1>(a, back, blocks, s);
    case 64 * 16 + 2: return norm_go<NX, NB, 64, 2>(a, back, blocks, s);
    case 64 * 16 + 4: return norm_go<NX, NB, 64, 4>(a, back, blocks, s);
    case 256 * 16 + 2: return norm_go<NX, NB, 256, 2>(a, back, blocks, s);
    case 256 * 16 + 4: return norm_go<NX, NB, 256, 4>(a, back, blocks, s);
    case 512 * 16 + 4: return norm_go<NX, NB, 512, 4>(a, back, blocks, s);
  }
  return DPVO_E_UNSUPPORTED;
}

}  // namespace
}  // namespace blk
