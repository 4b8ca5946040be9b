// blocks_dev.h -- what the gated feed-forward / residual-norm kernels (blocks_gemm.h, blocks_norm.h, blocks.hip) share: the three element
// types, loads and stores that end at a row's end, the activations and their derivatives.  Sums, statistics and activations are f32 throughout.
#pragma once
#include "common.h"
#include "blocks_plan.h"

#define BLK_INLINE __attribute__((always_inline))      // for lambdas: one that stays a call keeps its captures in scratch

namespace blk {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef int i4v __attribute__((ext_vector_type(4)));
typedef int i2v __attribute__((ext_vector_type(2)));

// 16 bytes of a row: KE elements
template <class T> struct Type { static constexpr int KE = 16 / (int)sizeof(T); };

// `memcpy` loads and stores: rows of odd length start at any element, and global memory is read in 16-byte pieces from any
// element's address (gfx950 has unaligned access switched on; an aligned address costs what an aligned load costs).
template <class V> __device__ __forceinline__ V ld_any(const void* p) {
  V v;
  __builtin_memcpy(&v, p, sizeof(V));
  return v;
}
template <class V> __device__ __forceinline__ void st_any(void* p, V v) { __builtin_memcpy(p, &v, sizeof(V)); }

// N consecutive elements as f32, of which `nv` (<= N) exist; the others read as 0 and are not touched
template <class T, int N> __device__ __forceinline__ void load_n(const T* p, int nv, float (&o)[N]) {
  if (nv >= N) {
    T t[N];
    __builtin_memcpy(t, p, sizeof(T) * N);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = (float)t[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = i < nv ? (float)p[i] : 0.f;
  }
}
template <class T, int N> __device__ __forceinline__ void store_n(T* p, int nv, const float (&v)[N]) {
  if (nv >= N) {
    T t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = (T)v[i];
    __builtin_memcpy(p, t, sizeof(T) * N);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < nv) p[i] = (T)v[i];
  }
}

// ---- activations.  FINE: expf / tanhf / division, for f32 results (f32 operands, and a 16-bit gate beside an f32 stream); otherwise the hardware
// exponential and reciprocal, whose error (2^-23 of |z| and a few 2^-22) is far below the half step of a 16-bit result (2^-11 / 2^-8).
template <bool FINE> __device__ __forceinline__ float exp_(float x) { return FINE ? expf(x) : __expf(x); }
template <bool FINE> __device__ __forceinline__ float rcp_(float x) { return FINE ? 1.f / x : __builtin_amdgcn_rcpf(x); }
template <bool FINE> __device__ __forceinline__ float sigmoid_(float x) { return rcp_<FINE>(1.f + exp_<FINE>(-x)); }
template <bool FINE> __device__ __forceinline__ float tanh_(float x) {
  if constexpr (FINE) return tanhf(x);
  return 1.f - 2.f * rcp_<FINE>(1.f + __expf(2.f * x));  // x -> +-inf: exp -> inf / 0, result -> +-1
}

template <bool FINE> __device__ __forceinline__ float act_(int a, float z) {
  switch (a) {
    case DPVO_ACT_RELU: return z < 0.f ? 0.f : z;                                    // (NaN stays NaN)
    case DPVO_ACT_SIGMOID: return sigmoid_<FINE>(z);
    case DPVO_ACT_SILU: return FINE ? z / (1.f + exp_<FINE>(-z)) : z * sigmoid_<FINE>(z);
    case DPVO_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    case DPVO_ACT_GELU_TANH: return 0.5f * z * (1.f + tanh_<FINE>(0.79788456080286536f * (z + 0.044715f * z * z * z)));
    default: return z;
  }
}
// value and derivative
struct ActD { float y, d; };
template <bool FINE> __device__ __forceinline__ ActD act_d(int a, float z) {
  switch (a) {
    case DPVO_ACT_RELU: return {z < 0.f ? 0.f : z, z <= 0.f ? 0.f : 1.f};          // (of a NaN as of a sum that may be positive: nothing is hidden)
    case DPVO_ACT_SIGMOID: { const float s = sigmoid_<FINE>(z); return {s, s * (1.f - s)}; }
    case DPVO_ACT_SILU: { const float s = sigmoid_<FINE>(z); return {z * s, s + z * (s * (1.f - s))}; }
    case DPVO_ACT_GELU: {
      const float c = 0.5f * (1.f + erff(z * 0.70710678118654752f));
      return {z * c, c + z * (0.39894228040143268f * exp_<FINE>(-0.5f * z * z))};
    }
    case DPVO_ACT_GELU_TANH: {
      const float t = tanh_<FINE>(0.79788456080286536f * (z + 0.044715f * z * z * z)), r = 1.f - t * t;
      // (r is 0 from |z| of some 5 on; z * z is infinite from 2^64 on, and the product would be a NaN)
      return {0.5f * z * (1.f + t), 0.5f * (1.f + t) + (r == 0.f ? 0.f : 0.5f * z * r * (0.79788456080286536f * (1.f + 0.134145f * z * z)))};
    }
    default: return {z, 1.f};
  }
}

// N at a time, the choice outside.  ALL: with the GELUs, whose polynomials' constants take some ninety registers inside a loop.
template <bool FINE, bool ALL, int N> __device__ __forceinline__ void act_n(int a, float (&v)[N]) {
#define BLK_CASE(A) case A: _Pragma("unroll") for (int e = 0; e < N; ++e) v[e] = act_<FINE>(A, v[e]); return;
  switch (a) {
    BLK_CASE(DPVO_ACT_RELU)
    BLK_CASE(DPVO_ACT_SIGMOID)
    BLK_CASE(DPVO_ACT_SILU)
  }
  if constexpr (ALL) switch (a) {
    BLK_CASE(DPVO_ACT_GELU)
    BLK_CASE(DPVO_ACT_GELU_TANH)
  }
#undef BLK_CASE
}
// z -> value y and derivative (in z)
template <bool FINE, bool ALL, int N> __device__ __forceinline__ void act_d_n(int a, float (&z)[N], float (&y)[N]) {
#define BLK_CASE(A) case A: _Pragma("unroll") for (int e = 0; e < N; ++e) { const ActD t = act_d<FINE>(A, z[e]); y[e] = t.y; z[e] = t.d; } return;
  switch (a) {
    BLK_CASE(DPVO_ACT_RELU)
    BLK_CASE(DPVO_ACT_SIGMOID)
    BLK_CASE(DPVO_ACT_SILU)
    BLK_CASE(DPVO_ACT_IDENTITY)
  }
  if constexpr (ALL) switch (a) {
    BLK_CASE(DPVO_ACT_GELU)
    BLK_CASE(DPVO_ACT_GELU_TANH)
  }
#undef BLK_CASE
}

// ---- the matrix products' arguments.  C[M,N] = sum over segments s of A_s . B_s, where an operand is stored either with the summed index
// contiguous ("row": A [M,K], B [N,K]) or with it as the row ("col": A [K,M], B [K,N]).
// E_LIN   out0 = act(C + bias0) + addend (save0: C + bias0 in f32); or, with `part`, the bare sum of this split in f32
// E_GATE  one A, two B: out0 = act(A.B0 + bias0) * (A.B1 + bias1) + addend (save0 / save1: the two sums in f32)
// E_GATE2 the same with an A for each B
// E_DACT  C is the gradient of h = act(save0) [* save1]: out0 = C [* save1] * act'(save0), out1 = C * act(save0) (with save1); with `mask`
//         (h itself, act = relu) out0 = C but where mask <= 0
struct Prob {
  const void *A[2], *B[2];
  int64_t lda[2], ldb[2], K[2];
  int64_t M, N;
  const void *bias0, *bias1, *addend, *mask;
  void *out0, *out1;
  void* colsum;                                          // F_TN: sums of A's columns [M], or with `part` their parts in f32
  float *save0, *save1, *part;
  int64_t ldadd, ldmask, ldo;
  int64_t tile0;                                         // first workgroup of this problem
  int64_t tm, tn;                                        // tiles
  int64_t nb0, nb;                                       // blocks of the summed index: first segment, all
  int splits, act;
};
struct GemmArgs {
  Prob p[MAXP];
  int n;
};

int gemm_f16(const GemmArgs& a, int form, int epi, int kind, int64_t tiles, hipStream_t s);
int gemm_bf16(const GemmArgs& a, int form, int epi, int kind, int64_t tiles, hipStream_t s);
int gemm_f32(const GemmArgs& a, int form, int epi, int kind, int64_t tiles, hipStream_t s);

}  // namespace blk
