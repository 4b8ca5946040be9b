// blocks.hip -- C entries of the gated feed-forward blocks and the norms around them (include/dpvo_hip.h), their small kernels, and the
// choice of tiles and splits.  The products themselves: blocks_gemm.h; the norms: blocks_norm.h.
#include <limits.h>
#include "blocks_dev.h"
#include "blocks_norm.h"

namespace blk {
namespace {

int gemm(const GemmArgs& a, int dtype, int form, int epi, int kind, int64_t tiles, hipStream_t s) {
  if (tiles > INT_MAX) return DPVO_E_UNSUPPORTED;
  if (dtype == DPVO_F16) return gemm_f16(a, form, epi, kind, tiles, s);
  if (dtype == DPVO_BF16) return gemm_bf16(a, form, epi, kind, tiles, s);
  return gemm_f32(a, form, epi, kind, tiles, s);
}

// out[e] = sum over parts of part[i][e] (+ bias[e % N]) (+ addend[e]), all contiguous; a job for each row of the grid
struct SumJob {
  const float* part;
  int64_t size;
  const void* addend;
  void* out;
  const void* bias;
  int64_t N;
};
struct SumArgs {
  SumJob j[2 * MAXP];
  int n, splits;
};
template <class T> __global__ void __launch_bounds__(256) split_sum_kernel(const SumArgs a) {
  const SumJob& j = ((const SumArgs*)__builtin_amdgcn_kernarg_segment_ptr())->j[blockIdx.y];
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (e >= j.size) return;
  const int nv = j.size - e < 4 ? (int)(j.size - e) : 4;
  float v[4] = {0.f, 0.f, 0.f, 0.f}, t[4];
  for (int s = 0; s < a.splits; ++s) {
    load_n<float, 4>(j.part + s * j.size + e, nv, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += t[i];
  }
  if (j.bias) {
    int64_t n = e % j.N;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < nv) v[i] += (float)((const T*)j.bias)[n];
      n = n + 1 < j.N ? n + 1 : 0;
    }
  }
  if (j.addend) {
    load_n<T, 4>((const T*)j.addend + e, nv, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += t[i];
  }
  store_n<T, 4>((T*)j.out + e, nv, v);
}
int split_sum(const SumArgs& a, int dtype, hipStream_t s) {
  int64_t size = 0;
  for (int i = 0; i < a.n; ++i) size = a.j[i].size > size ? a.j[i].size : size;
  if (size == 0) return DPVO_OK;
  const int64_t blocks = cdiv64(cdiv64(size, 4), 256);
  if (blocks > INT_MAX) return DPVO_E_UNSUPPORTED;
  const dim3 grid((unsigned)blocks, (unsigned)a.n);
  if (dtype == DPVO_F16) hipLaunchKernelGGL((split_sum_kernel<_Float16>), grid, dim3(256), 0, s, a);
  else if (dtype == DPVO_BF16) hipLaunchKernelGGL((split_sum_kernel<__bf16>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((split_sum_kernel<float>), grid, dim3(256), 0, s, a);
  DPVO_LAUNCH_CHECK();
  return DPVO_OK;
}

// dpvo_gated_linear_dact: one pass, 8 elements a thread; 45312 x 384 in f16 45 us, 244 MB at 5.4 TB/s
template <class T> __global__ void __launch_bounds__(256) dact_kernel(const T* dy, int64_t lddy, const float* gate, const float* up, T* dg, T* du, int64_t ldo,
                                                                       int act, int64_t M, int64_t N) {
  const int64_t n8 = (N + 7) / 8, total = M * n8;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / n8, n = (i % n8) * 8;
    const int nv = N - n < 8 ? (int)(N - n) : 8;
    float d[8], g[8], u[8];
    load_n<T, 8>(dy + m * lddy + n, nv, d);
    load_n<float, 8>(gate + m * N + n, nv, g);
    if (up) load_n<float, 8>(up + m * N + n, nv, u);
    float o[8];
    act_d_n<sizeof(T) == 4, true>(act, g, o);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      o[e] *= d[e];
      d[e] *= up ? u[e] * g[e] : g[e];
    }
    store_n<T, 8>(dg + m * ldo + n, nv, d);
    if (up) store_n<T, 8>(du + m * ldo + n, nv, o);
  }
}

// ---- partial rows -> rows
struct ColJob {
  float* part;
  void* out;
  int64_t N;
  int64_t parts;                                         // partial rows to one output row
  int64_t outs;                                          // output rows
  int type;                                              // of `out`
};
struct ColArgs {
  ColJob j[5];
  int n;
};
// out[o][c] = sum of part[o * parts + p][c]: 64 columns x 16 shares of the partial rows, eight loads of each under way
__global__ void __launch_bounds__(1024) col_reduce_kernel(const ColArgs) {
  __shared__ float lds[16][64];
  const ColJob& j = ((const ColArgs*)__builtin_amdgcn_kernarg_segment_ptr())->j[blockIdx.z];
  const int64_t c0 = (int64_t)blockIdx.x * 64, c = c0 + threadIdx.x % 64;
  const int share = threadIdx.x / 64;
  if (c0 >= j.N) return;
  for (int64_t o = blockIdx.y; o < j.outs; o += gridDim.y) {
    float s = 0.f;
    if (c < j.N) {
      const float* q = j.part + o * j.parts * j.N + c;
      int64_t p = share;
      for (; p + 7 * 16 < j.parts; p += 8 * 16) {
        float t[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) t[k] = q[(p + k * 16) * j.N];
#pragma unroll
        for (int k = 0; k < 8; ++k) s += t[k];
      }
      for (; p < j.parts; p += 16) s += q[p * j.N];
    }
    lds[share][threadIdx.x % 64] = s;
    __syncthreads();
    if (threadIdx.x < 64 && c < j.N) {
      s = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) s += lds[k][threadIdx.x];
      if (j.type == DPVO_F16) ((_Float16*)j.out)[o * j.N + c] = (_Float16)s;
      else if (j.type == DPVO_BF16) ((__bf16*)j.out)[o * j.N + c] = (__bf16)s;
      else ((float*)j.out)[o * j.N + c] = s;
    }
    __syncthreads();
  }
}
int col_reduce(const ColArgs& c, hipStream_t s) {
  if (c.n == 0) return DPVO_OK;
  int64_t w = 0, o = 0;
  for (int i = 0; i < c.n; ++i) {
    w = c.j[i].N > w ? c.j[i].N : w;
    o = c.j[i].outs > o ? c.j[i].outs : o;
  }
  if (w == 0 || o == 0) return DPVO_OK;
  hipLaunchKernelGGL(col_reduce_kernel, dim3((unsigned)cdiv64(w, 64), (unsigned)(o < 1024 ? o : 1024), (unsigned)c.n), dim3(1024), 0, s, c);
  DPVO_LAUNCH_CHECK();
  return DPVO_OK;
}
int64_t tiles_of(Prob& p, int kind, int halves = 1) {
  const int t = tile_size(kind);
  p.tm = cdiv64(p.M, t);
  p.tn = cdiv64(p.N, t / halves);
  return p.tm * p.tn;
}

int norm_check(const dpvo_residual_norm_t* p) {
  if (!p || p->M < 0 || p->D < 1 || !type_ok(p->x_dtype) || !type_ok(p->f_dtype) || !type_ok(p->w_dtype)) return DPVO_E_INVALID;
  if (p->x_dtype != p->f_dtype && p->x_dtype != DPVO_F32) return DPVO_E_UNSUPPORTED;
  if (p->h_dtype != p->x_dtype && p->h_dtype != p->f_dtype) return DPVO_E_UNSUPPORTED;
  if (p->norm < DPVO_NORM_NONE || p->norm > DPVO_NORM_RMS || p->post < DPVO_NORM_NONE || p->post > DPVO_NORM_RMS) return DPVO_E_INVALID;
  if (!act_ok(p->gate_activation)) return DPVO_E_INVALID;
  if (p->gate_activation > DPVO_ACT_SILU) return DPVO_E_UNSUPPORTED;
  if (p->D > NORM_MAX_D || p->M > INT_MAX) return DPVO_E_UNSUPPORTED;
  if (p->gate && p->M && (!p->f || p->groups < 1 || p->M % p->groups)) return DPVO_E_INVALID;
  if (p->M && !p->x) return DPVO_E_INVALID;
  return DPVO_OK;
}
int norm_run(const NormArgs& a, int sh, bool back, int64_t blocks, hipStream_t s) {
  if (a.p.f_dtype == DPVO_F16) return norm_f16(a, sh, back, blocks, s);
  if (a.p.f_dtype == DPVO_BF16) return norm_bf16(a, sh, back, blocks, s);
  return norm_f32(a, sh, back, blocks, s);
}

}  // namespace
}  // namespace blk

using namespace blk;

extern "C" size_t dpvo_gated_linear_workspace_bytes(const dpvo_gated_linear_t* p) {
  if (!p || !type_ok(p->dtype) || p->M <= 0 || p->N <= 0 || p->K < 0 || p->Kv < 0 || p->w_up) return 0;
  if (linear_few(p, E_LIN)) return 0;
  const Plan c = linear_plan(p, E_LIN);
  return c.splits > 1 ? (size_t)(c.splits * p->M * p->N * 4) : 0;
}

extern "C" int dpvo_gated_linear(const dpvo_gated_linear_t* p, void* ws, size_t ws_bytes, void* stream) {
  if (!p || !type_ok(p->dtype) || !act_ok(p->activation) || p->M < 0 || p->N < 0 || p->K < 0 || p->Kv < 0) return DPVO_E_INVALID;
  if (p->M == 0 || p->N == 0) return DPVO_OK;
  const int size = type_size(p->dtype);
  if (!p->y || (p->K && (!p->x || !p->w_gate)) || (p->w_up && p->Kv && !p->v)) return DPVO_E_INVALID;
  if (!ld_ok(p->ldx, p->K, size) || !ld_ok(p->ldwg, p->K, size) || p->ldy < p->N || (p->residual && p->ldr < p->N)) return DPVO_E_INVALID;
  if (p->w_up && (!ld_ok(p->ldv, p->Kv, size) || !ld_ok(p->ldwu, p->Kv, size))) return DPVO_E_INVALID;
  hipStream_t s = (hipStream_t)stream;
  const int bk = block_k(p->dtype), epi = linear_epi(p);
  GemmArgs a = {};
  a.n = 1;
  Prob& q = a.p[0];
  q.A[0] = p->x; q.B[0] = p->w_gate; q.lda[0] = p->ldx; q.ldb[0] = p->ldwg; q.K[0] = p->K;
  q.A[1] = p->v; q.B[1] = p->w_up; q.lda[1] = p->ldv; q.ldb[1] = p->ldwu; q.K[1] = p->Kv;
  q.M = p->M; q.N = p->N;
  q.bias0 = p->b_gate; q.bias1 = p->b_up; q.addend = p->residual; q.ldadd = p->ldr;
  q.out0 = p->y; q.ldo = p->ldy; q.save0 = p->save_gate; q.save1 = p->w_up ? p->save_up : nullptr;
  q.act = p->activation; q.splits = 1;
  q.nb0 = cdiv64(p->K, bk);
  q.nb = q.nb0 + (epi == E_GATE2 ? cdiv64(p->Kv, bk) : 0);
  if (linear_few(p, epi)) return gemm(a, p->dtype, F_NT, epi, T_FEW, cdiv64(p->N, 16), s);
  const Plan c = linear_plan(p, epi);
  const int64_t n = tiles_of(q, c.kind, epi == E_GATE ? 2 : 1);
  if (c.splits == 1) return gemm(a, p->dtype, F_NT, epi, c.kind, n, s);
  if ((size_t)(c.splits * p->M * p->N * 4) > ws_bytes || !ws) return DPVO_E_WORKSPACE;
  q.splits = (int)c.splits;
  q.part = (float*)ws;
  const int rc = gemm(a, p->dtype, F_NT, epi, c.kind, n * c.splits, s);
  SumArgs sum = {};
  sum.n = 1;
  sum.splits = q.splits;
  sum.j[0] = {q.part, p->M * p->N, p->residual, p->y, p->b_gate, p->N};
  return rc ? rc : split_sum(sum, p->dtype, s);
}

extern "C" int dpvo_gated_linear_dact(const void* dy, int64_t lddy, const float* gate, const float* up, void* d_gate, void* d_up, int64_t ldo, int dtype,
                                      int activation, int64_t M, int64_t N, void* stream) {
  if (!type_ok(dtype) || !act_ok(activation) || M < 0 || N < 0) return DPVO_E_INVALID;
  if (M == 0 || N == 0) return DPVO_OK;
  if (!dy || !gate || !d_gate || (up && !d_up) || lddy < N || ldo < N) return DPVO_E_INVALID;
  const int64_t want = cdiv64(M * cdiv64(N, 8), 256), blocks = want < 16384 ? want : 16384;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DPVO_F16) hipLaunchKernelGGL((dact_kernel<_Float16>), dim3((unsigned)blocks), dim3(256), 0, s, (const _Float16*)dy, lddy, gate, up, (_Float16*)d_gate, (_Float16*)d_up, ldo, activation, M, N);
  else if (dtype == DPVO_BF16) hipLaunchKernelGGL((dact_kernel<__bf16>), dim3((unsigned)blocks), dim3(256), 0, s, (const __bf16*)dy, lddy, gate, up, (__bf16*)d_gate, (__bf16*)d_up, ldo, activation, M, N);
  else hipLaunchKernelGGL((dact_kernel<float>), dim3((unsigned)blocks), dim3(256), 0, s, (const float*)dy, lddy, gate, up, (float*)d_gate, (float*)d_up, ldo, activation, M, N);
  DPVO_LAUNCH_CHECK();
  return DPVO_OK;
}

extern "C" size_t dpvo_gated_linear_dx_workspace_bytes(const dpvo_gated_linear_dx_t* p) {
  if (!p || !type_ok(p->dtype) || p->M <= 0 || p->N <= 0 || p->K[0] < 0 || p->K[1] < 0 || p->gate || p->mask) return 0;
  if (p->lddx != p->N || (p->addend && p->ldadd != p->N)) return 0;
  const int bk = block_k(p->dtype);
  const Plan c = dx_plan(p->M, p->N, cdiv64(p->K[0], bk) + (p->a[1] ? cdiv64(p->K[1], bk) : 0), p->dtype, true);
  return c.splits > 1 ? (size_t)(c.splits * p->M * p->N * 4) : 0;
}

extern "C" int dpvo_gated_linear_dx(const dpvo_gated_linear_dx_t* p, void* ws, size_t ws_bytes, void* stream) {
  if (!p || !type_ok(p->dtype) || !act_ok(p->activation) || p->M < 0 || p->N < 0 || p->K[0] < 0 || p->K[1] < 0) return DPVO_E_INVALID;
  if (p->M == 0 || p->N == 0) return DPVO_OK;
  const int size = type_size(p->dtype), bk = block_k(p->dtype);
  if (!p->dx || p->lddx < p->N || (p->addend && p->ldadd < p->N) || (p->mask && p->ldmask < p->N)) return DPVO_E_INVALID;
  if ((p->gate || p->mask) && p->addend) return DPVO_E_UNSUPPORTED;
  if ((p->gate && p->mask) || (p->up && (!p->gate || !p->dx2))) return DPVO_E_INVALID;
  const int64_t K1 = p->a[1] ? p->K[1] : 0;
  for (int i = 0; i < 2; ++i) {
    const int64_t k = i ? K1 : p->K[0];
    if (k && (!p->a[i] || !p->b[i])) return DPVO_E_INVALID;
    if (k && (!ld_ok(p->lda[i], k, size) || !ld_ok(p->ldb[i], p->N, size))) return DPVO_E_INVALID;
  }
  GemmArgs a = {};
  a.n = 1;
  Prob& q = a.p[0];
  for (int i = 0; i < 2; ++i) {
    q.A[i] = p->a[i]; q.B[i] = p->b[i]; q.lda[i] = p->lda[i]; q.ldb[i] = p->ldb[i];
  }
  q.K[0] = p->K[0]; q.K[1] = K1;
  q.M = p->M; q.N = p->N;
  q.out0 = p->dx; q.out1 = p->dx2; q.ldo = p->lddx; q.act = p->activation;
  q.nb0 = cdiv64(p->K[0], bk);
  q.nb = q.nb0 + cdiv64(K1, bk);
  q.splits = 1;
  hipStream_t s = (hipStream_t)stream;
  if (p->gate || p->mask) {
    const int kind = dx_plan(p->M, p->N, q.nb, p->dtype, false).kind;
    tiles_of(q, kind);
    q.save0 = (float*)p->gate; q.save1 = (float*)p->up; q.mask = p->mask; q.ldmask = p->ldmask;
    return gemm(a, p->dtype, F_NN, E_DACT, kind, q.tm * q.tn, s);
  }
  q.act = DPVO_ACT_IDENTITY;
  const bool flat = p->lddx == p->N && (!p->addend || p->ldadd == p->N);
  const Plan c = dx_plan(p->M, p->N, q.nb, p->dtype, flat);
  tiles_of(q, c.kind);
  if (c.splits > 1) {
    if ((size_t)(c.splits * p->M * p->N * 4) > ws_bytes || !ws) return DPVO_E_WORKSPACE;
    q.splits = (int)c.splits;
    q.part = (float*)ws;
    const int rc = gemm(a, p->dtype, F_NN, E_LIN, c.kind, q.tm * q.tn * c.splits, s);
    SumArgs sum = {};
    sum.n = 1;
    sum.splits = q.splits;
    sum.j[0] = {q.part, p->M * p->N, p->addend, p->dx, nullptr, 0};
    return rc ? rc : split_sum(sum, p->dtype, s);
  }
  q.addend = p->addend; q.ldadd = p->ldadd;
  return gemm(a, p->dtype, F_NN, E_LIN, c.kind, q.tm * q.tn, s);
}

// workspace: the parts of each product and of its column sums
static bool dw_ok(const dpvo_gated_linear_dw_t* p) {
  if (!p || p->n < 0 || p->n > MAXP || !type_ok(p->dtype) || p->M < 0) return false;
  for (int i = 0; i < p->n; ++i) {
    if (p->N[i] < 0 || p->K[i] < 0) return false;
    if (!p->N[i]) continue;
    if (p->K[i] ? !p->dw[i] : p->db[i] != nullptr) return false;
    if (!p->M) continue;
    if (!p->a[i] || !ld_ok(p->lda[i], p->N[i], type_size(p->dtype))) return false;
    if (p->K[i] && (!p->b[i] || !ld_ok(p->ldb[i], p->K[i], type_size(p->dtype)))) return false;
  }
  return true;
}
extern "C" size_t dpvo_gated_linear_dw_workspace_bytes(const dpvo_gated_linear_dw_t* p) {
  if (!dw_ok(p)) return 0;
  const int64_t s = dw_plan(p).splits;
  int64_t f = 0;
  for (int i = 0; i < p->n; ++i) {
    if (s > 1) f += s * p->N[i] * (p->K[i] + (p->db[i] != nullptr));
  }
  return (size_t)f * 4;
}
extern "C" int dpvo_gated_linear_dw(const dpvo_gated_linear_dw_t* p, void* ws, size_t ws_bytes, void* stream) {
  if (!dw_ok(p)) return DPVO_E_INVALID;
  const size_t need = dpvo_gated_linear_dw_workspace_bytes(p);
  if (need > ws_bytes || (need && !ws)) return DPVO_E_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  const Plan c0 = dw_plan(p);
  const int64_t splits = c0.splits;
  float* w = (float*)ws;
  GemmArgs a = {};
  int64_t n = 0;
  SumArgs sum = {};
  sum.splits = (int)splits;
  for (int i = 0; i < p->n; ++i) {
    if (!p->N[i] || !p->K[i]) continue;
    Prob& q = a.p[a.n++];
    q.A[0] = p->a[i]; q.B[0] = p->b[i]; q.lda[0] = p->lda[i]; q.ldb[0] = p->ldb[i]; q.K[0] = p->M;
    q.M = p->N[i]; q.N = p->K[i];
    q.nb0 = q.nb = cdiv64(p->M, block_k(p->dtype));
    q.splits = (int)splits;
    q.out0 = p->dw[i]; q.ldo = p->K[i]; q.colsum = p->db[i];
    if (splits > 1) {
      sum.j[sum.n++] = {q.part = w, q.M * q.N, nullptr, p->dw[i], nullptr, 0};
      w += splits * q.M * q.N;
      if (p->db[i]) {
        sum.j[sum.n++] = {w, q.M, nullptr, p->db[i], nullptr, 0};
        q.colsum = w;
        w += splits * q.M;
      }
    }
    q.tile0 = n;
    n += tiles_of(q, c0.kind) * splits;
  }
  const int rc = gemm(a, p->dtype, F_TN, E_LIN, c0.kind, n, s);
  return rc || splits == 1 ? rc : split_sum(sum, p->dtype, s);
}

extern "C" int dpvo_residual_norm(const dpvo_residual_norm_t* p, void* stream) {
  const int rc = norm_check(p);
  if (rc) return rc;
  if (p->M == 0) return DPVO_OK;
  if (p->ldx < p->D || (p->f && p->ldf < p->D) || (p->gate && p->ldgate < p->D) || (p->norm && !p->h) || (!p->norm && !p->s)) return DPVO_E_INVALID;
  NormArgs a = {};
  a.p = *p;
  a.rows_per_gate = p->gate ? (uint32_t)(p->M / p->groups) : 1;
  const int sh = norm_shape(*p, false, 0);
  // Ragged rows profit from several to a workgroup, whose loads then run ahead: `norm` of 4096 x 2333 bf16 27 us with 2048 workgroups, 35 with 8192,
  // 45312 x 385 27 and 42, f32 29 and 39.  Rows of whole pieces: with two inputs in f32 8192 loses nothing and 2048 up to 8 % (45312 x 384 51 and 55 us,
  // 16384 x 4000 194 and 201); in 16 bits 2048 would be faster, by 8 to 24 % for `norm` alone (8192 x 4096 38 and 31 us) and 0 to 10 % with a branch.
  const int64_t want = cdiv64(p->M, norm_slots(sh)), most = p->D % 8 ? 2048 : 8192;
  return norm_run(a, sh, false, want < most ? want : most, (hipStream_t)stream);
}

extern "C" size_t dpvo_residual_norm_backward_workspace_bytes(const dpvo_residual_norm_t* p) {
  if (norm_check(p) || p->M == 0) return 0;
  const NormPlan n = norm_plan(*p);
  const int64_t rows = (n.shared && p->dgate ? n.groups * n.bpg : 0) + n.blocks * ((p->dw != nullptr) + (p->db != nullptr) + (p->dpw != nullptr) + (p->dpb != nullptr));
  return (size_t)(rows * p->D * 4 + (n.sh == NORM_WIDE && rows ? p->M * NORM_STATS * 4 : 0));
}
extern "C" int dpvo_residual_norm_backward(const dpvo_residual_norm_t* p, void* ws, size_t ws_bytes, void* stream) {
  int rc = norm_check(p);
  if (rc) return rc;
  if (p->ldx < p->D || (p->f && p->ldf < p->D) || (p->gate && p->ldgate < p->D) || (p->ds && p->ldds < p->D) || (p->dh && p->lddh < p->D)) return DPVO_E_INVALID;
  if ((!p->f && (p->df || p->dgate || p->dpw || p->dpb)) || (p->dgate && !p->gate) || (p->post == DPVO_NORM_NONE && (p->dpw || p->dpb))) return DPVO_E_INVALID;
  const size_t need = dpvo_residual_norm_backward_workspace_bytes(p);
  if (need > ws_bytes || (need && !ws)) return DPVO_E_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  NormArgs a = {};
  a.p = *p;
  ColArgs c = {};
  float* w = (float*)ws;
  const NormPlan n = p->M ? norm_plan(*p) : NormPlan{0, 0, 0, 1, 1, 0, false};
  a.shared = n.shared;
  a.groups = n.groups; a.rpg = n.rpg; a.gpb = n.gpb; a.bpg = n.bpg;
  auto job = [&](void* out, int type, int64_t outs, int64_t parts) {
    if (!out) return (float*)nullptr;
    ColJob& j = c.j[c.n++];
    j.part = w; j.out = out; j.type = type; j.N = p->D; j.outs = outs; j.parts = parts;
    w += outs * parts * p->D;
    return j.part;
  };
  a.part_w = job(p->dw, p->w_dtype, 1, n.blocks);
  a.part_b = job(p->db, p->w_dtype, 1, n.blocks);
  a.part_pw = job(p->dpw, p->w_dtype, 1, n.blocks);
  a.part_pb = job(p->dpb, p->w_dtype, 1, n.blocks);
  if (n.shared) a.part_gate = job(p->dgate, p->f_dtype, n.groups, n.bpg);
  else if (!p->M && p->dgate) job(p->dgate, p->f_dtype, p->groups, 0);
  if (n.sh == NORM_WIDE && c.n) a.stats = w;
  if (p->M) {
    rc = norm_run(a, n.sh, true, n.blocks, s);
    if (rc) return rc;
  }
  return col_reduce(c, s);                               // (no rows: parts = 0, the shared gradients are zeros)
}
