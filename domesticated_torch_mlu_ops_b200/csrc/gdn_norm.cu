// Gated RMS norm with residual sum, and its gradient.
//   r = residual + alpha x                       (r = x without a residual)
//   u = r act(z) when the gate comes before the norm, else r
//   n = u rstd,  rstd = (mean of u^2 over a group + eps)^-1/2
//   y = n w, then times act(z) when the gate comes after the norm
// and with g = dy act(z) (gate after) or dy, dn = g w, c = mean(dn n):
//   du = rstd (dn - n c);  dr = du (gate before: du act(z)) + dsum
//   dw = sum over rows of g n;  dz = dy n w act'(z) or du r act'(z)
//   dx = alpha dr, dresidual = dr
//
// Both passes are streams: each input is read once and each output written
// once, so HBM bounds them.  A row's group stays in the registers of a team
// of threads between its reduction and its outputs: 8, 16 or 32 lanes of a
// warp (several teams per warp share its reductions) up to 128 vectors, a
// whole CTA above.  The backward recomputes rstd (one more value in a
// reduction that it needs anyway) instead of reading a saved one; its teams
// walk the rows of one group with dw in registers, CTAs leave their dw in
// the workspace and a second kernel adds those in order.

#include "conv_math.cuh"
#include "gdn_common.cuh"
#include "gdn_internal.h"

#include <algorithm>

namespace gdn {
namespace norm {

using conv::ld_any;
using conv::ldv;
using conv::st_any;
using conv::stv;

struct Params {
  const void* x;  // forward: T; backward: X
  const void* z;
  const void* residual;
  const void* weight;
  void* y;
  void* sum;
  const void *dy, *dsum;
  void *dx, *dz, *dresidual;
  float* partial;  // [gridDim.x][D]
  int64_t rows, heads, D;
  int64_t sx_tok, sx_head, sz_tok, sz_head;  // row (t, h) of x and z, in elements
  int group;
  int w_dtype, res_f32, gate_before, sigmoid_gate;
  float eps, alpha, w_off;
};

// act(z) and act'(z), with the hardware exponential and divide.
__device__ __forceinline__ float gate(float z, int sigmoid_gate) {
  const float s = __fdividef(1.f, 1.f + __expf(-z));
  return sigmoid_gate ? s : z * s;
}
__device__ __forceinline__ void gate_grad(float z, int sigmoid_gate, float& a, float& da) {
  const float s = __fdividef(1.f, 1.f + __expf(-z));
  a = sigmoid_gate ? s : z * s;
  da = sigmoid_gate ? s * (1.f - s) : s * fmaf(z, 1.f - s, 1.f);
}

// VEC values as floats from T or fp32 rows (fp32 vectors of 8 as two 16-byte loads).
template <int VEC>
__device__ __forceinline__ void ldf(const float* p, float* v) {
  if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(p + i));
      v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = __ldg(p + i);
  }
}
template <int VEC>
__device__ __forceinline__ void stf(float* p, const float* v) {
  if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) p[i] = v[i];
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void ld_res(const void* p, int f32, int64_t i, float* v) {
  if (f32) ldf<VEC>(static_cast<const float*>(p) + i, v);
  else ldv<T, VEC>(static_cast<const T*>(p) + i, v);
}
template <typename T, int VEC>
__device__ __forceinline__ void st_res(void* p, int f32, int64_t i, const float* v) {
  if (f32) stf<VEC>(static_cast<float*>(p) + i, v);
  else stv<T, VEC>(static_cast<T*>(p) + i, v);
}
template <int VEC>
__device__ __forceinline__ void ld_weight(const Params& p, int64_t i, float* w) {
  if (VEC > 1 && p.w_dtype == GDN_F32) {
    ldf<VEC>(static_cast<const float*>(p.weight) + i, w);
  } else if (VEC > 1 && p.w_dtype == GDN_BF16) {
#pragma unroll
    for (int e = 0; e < VEC; e += 4) {
      const float4 f = load4(static_cast<const __nv_bfloat16*>(p.weight) + i + e);
      w[e] = f.x; w[e + 1] = f.y; w[e + 2] = f.z; w[e + 3] = f.w;
    }
  } else if (VEC > 1) {
#pragma unroll
    for (int e = 0; e < VEC; e += 4) {
      const float4 f = load4(static_cast<const __half*>(p.weight) + i + e);
      w[e] = f.x; w[e + 1] = f.y; w[e + 2] = f.z; w[e + 3] = f.w;
    }
  } else {
    w[0] = ld_any(p.weight, p.w_dtype, i);
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) w[e] += p.w_off;
}

// Sum over the team: TS lanes of a warp, or (TS = 0) the CTA; `buf` holds
// one value per warp and alternates between calls.
template <int TS, int K>
__device__ __forceinline__ void team_sum(float* v, float (*buf)[32]) {
#pragma unroll
  for (int o = (TS ? TS : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (TS == 0) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    if (lane == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) buf[k][warp] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float a = lane < nw ? buf[k][lane] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
      v[k] = a;
    }
  }
}

// One team per (row, group).  TS = 0: the CTA.
template <typename T, int VEC, int ITER, int TS, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_fwd_kernel(const Params p) {
  __shared__ float buf[1][32];
  const int ts = TS ? TS : blockDim.x;
  const int lane = TS ? threadIdx.x % TS : threadIdx.x;
  const int64_t teams = blockDim.x / ts;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * teams + (TS ? threadIdx.x / TS : 0);
  const int64_t g0 = static_cast<int64_t>(blockIdx.y) * p.group;
  const bool live = row < p.rows;  // every lane stays for the shuffles
  const int64_t tok = live ? row / p.heads : 0, head = live ? row - tok * p.heads : 0;
  const T* x = static_cast<const T*>(p.x) + tok * p.sx_tok + head * p.sx_head + g0;
  const T* z = p.z ? static_cast<const T*>(p.z) + tok * p.sz_tok + head * p.sz_head + g0 : nullptr;
  float u[ITER][VEC], a[ITER][VEC];
  float ss[1] = {0.f};
#pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const int i = (k * ts + lane) * VEC;
    const bool in = live && i < p.group;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      u[k][e] = 0.f;
      a[k][e] = 0.f;
    }
    if (in) {
      ldv<T, VEC>(x + i, u[k]);
      if (z) ldv<T, VEC>(z + i, a[k]);
      if (p.residual) {
        float r[VEC];
        ld_res<T, VEC>(p.residual, p.res_f32, row * p.D + g0 + i, r);
#pragma unroll
        for (int e = 0; e < VEC; ++e) u[k][e] = fmaf(p.alpha, u[k][e], r[e]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const int i = (k * ts + lane) * VEC;
    if (p.sum && live && i < p.group) st_res<T, VEC>(p.sum, p.res_f32, row * p.D + g0 + i, u[k]);
    if (z)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        a[k][e] = gate(a[k][e], p.sigmoid_gate);
        if (p.gate_before) u[k][e] = i < p.group ? u[k][e] * a[k][e] : 0.f;
      }
#pragma unroll
    for (int e = 0; e < VEC; ++e) ss[0] = fmaf(u[k][e], u[k][e], ss[0]);
  }
  team_sum<TS, 1>(ss, buf);
  const float rstd = rsqrtf(ss[0] / static_cast<float>(p.group) + p.eps);
  if (!live) return;
  const bool after = z && !p.gate_before;
#pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const int i = (k * ts + lane) * VEC;
    if (i >= p.group) break;
    float w[VEC];
    ld_weight<VEC>(p, g0 + i, w);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      u[k][e] = u[k][e] * rstd * w[e];
      if (after) u[k][e] *= a[k][e];
    }
    stv<T, VEC>(static_cast<T*>(p.y) + row * p.D + g0 + i, u[k]);
  }
}

// X: the type of x (the residual's when the forward summed one).  A team
// walks rows blockIdx.x * teams + team, + gridDim.x * teams, ...
template <typename T, typename X, int VEC, int ITER, int TS, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_bwd_kernel(const Params p) {
  extern __shared__ float dws[];  // [teams][group] when teams > 1
  __shared__ float buf[2][2][32];
  const int ts = TS ? TS : blockDim.x;
  const int lane = TS ? threadIdx.x % TS : threadIdx.x;
  const int team = TS ? threadIdx.x / TS : 0;
  const int64_t teams = blockDim.x / ts;
  const int64_t g0 = static_cast<int64_t>(blockIdx.y) * p.group;
  const float inv = 1.f / static_cast<float>(p.group);
  float w[ITER][VEC], dw[ITER][VEC];
#pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const int i = (k * ts + lane) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[k][e] = 0.f;
      dw[k][e] = 0.f;
    }
    if (i < p.group) ld_weight<VEC>(p, g0 + i, w[k]);
  }
  int par = 0;
  // the CTA's teams walk together (shuffles and barriers are for all of them)
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * teams; row0 < p.rows; row0 += gridDim.x * teams) {
    const int64_t row = row0 + team;
    const bool live = row < p.rows;
    const int64_t tok = live ? row / p.heads : 0, head = live ? row - tok * p.heads : 0;
    const X* x = static_cast<const X*>(p.x) + tok * p.sx_tok + head * p.sx_head + g0;
    const T* z = p.z ? static_cast<const T*>(p.z) + tok * p.sz_tok + head * p.sz_head + g0 : nullptr;
    const int64_t at = row * p.D + g0;
    float r[ITER][VEC], d[ITER][VEC], zz[ITER][VEC];
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      const int i = (k * ts + lane) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        r[k][e] = 0.f;
        d[k][e] = 0.f;
        zz[k][e] = 0.f;
      }
      if (live && i < p.group) {
        if constexpr (sizeof(X) == 4) ldf<VEC>(x + i, r[k]);
        else ldv<X, VEC>(x + i, r[k]);
        ldv<T, VEC>(static_cast<const T*>(p.dy) + at + i, d[k]);
        if (z) ldv<T, VEC>(z + i, zz[k]);
      }
    }
    float s[2] = {0.f, 0.f};  // sum u^2, sum dn u
#pragma unroll
    for (int k = 0; k < ITER; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float u = r[k][e], g = d[k][e];
        if (z) {
          const float a = gate(zz[k][e], p.sigmoid_gate);
          if (p.gate_before) u *= a;
          else g *= a;
        }
        s[0] = fmaf(u, u, s[0]);
        s[1] = fmaf(g * w[k][e], u, s[1]);
      }
    team_sum<TS, 2>(s, buf[par]);
    par ^= 1;
    const float rstd = rsqrtf(s[0] * inv + p.eps);
    const float c = s[1] * rstd * inv;  // mean(dn n)
    if (!live) continue;
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      const int i = (k * ts + lane) * VEC;
      if (i >= p.group) break;
      float dr[VEC], dz[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float a = 1.f, da = 0.f;
        if (z) gate_grad(zz[k][e], p.sigmoid_gate, a, da);
        const float u = p.gate_before ? r[k][e] * a : r[k][e];
        const float n = u * rstd;
        const float g = p.gate_before ? d[k][e] : d[k][e] * a;
        dw[k][e] = fmaf(g, n, dw[k][e]);
        const float du = rstd * fmaf(-n, c, g * w[k][e]);
        dz[e] = (p.gate_before ? du * r[k][e] : d[k][e] * n * w[k][e]) * da;
        dr[e] = p.gate_before ? du * a : du;
      }
      if (z) stv<T, VEC>(static_cast<T*>(p.dz) + at + i, dz);
      if (p.dsum) {
        float ds[VEC];
        ld_res<T, VEC>(p.dsum, p.res_f32, at + i, ds);
#pragma unroll
        for (int e = 0; e < VEC; ++e) dr[e] += ds[e];
      }
      if (p.dresidual) st_res<T, VEC>(p.dresidual, p.res_f32, at + i, dr);
#pragma unroll
      for (int e = 0; e < VEC; ++e) dr[e] *= p.alpha;
      stv<T, VEC>(static_cast<T*>(p.dx) + at + i, dr);
    }
  }
  float* out = p.partial + static_cast<int64_t>(blockIdx.x) * p.D + g0;
  if (TS == 0) {
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      const int i = (k * ts + lane) * VEC;
      if (i < p.group) stf<1>(out + i, dw[k]);
#pragma unroll
      for (int e = 1; e < VEC; ++e)
        if (i < p.group) out[i + e] = dw[k][e];
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const int i = (k * ts + lane) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (i < p.group) dws[team * p.group + i + e] = dw[k][e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.group; i += blockDim.x) {
    float a = 0.f;
    for (int t = 0; t < teams; ++t) a += dws[t * p.group + i];
    out[i] = a;
  }
}

// dw = sum of the CTAs' parts, in order: 32 lanes of parts per column.
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float* partial, int64_t parts, int64_t D, void* dw,
                                                       int w_dtype) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  float acc = 0.f;
  if (c < D)
#pragma unroll 4
    for (int64_t s = row; s < parts; s += 32) acc += partial[s * D + c];
  part[row][lane] = acc;
  __syncthreads();
  // lane and row swap: warp `row` adds the 32 sums of column blockIdx.x * 32 + row
  float v = part[lane][row];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int64_t cc = static_cast<int64_t>(blockIdx.x) * 32 + row;
  if (lane == 0 && cc < D) st_any(dw, w_dtype, cc, v);
}

// ---- host ------------------------------------------------------------------
bool fdtype_ok(int d) { return d == GDN_F32 || d == GDN_BF16 || d == GDN_F16; }
int esize(int d) { return d == GDN_F32 ? 4 : 2; }
bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr int kMaxScalar = 16 * 1024, kMaxVector = 4 * 1024;  // elements / vectors a CTA can hold

// 16-byte vectors when the group, the strides and every pointer allow them.
int vec_of(const gdn_norm_args& a) {
  const int v = 16 / esize(a.x_dtype), xv = 16 / esize(a.x_dtype);
  const bool ok = a.group % v == 0 && a.D % v == 0 && a.stride_x_token % xv == 0 && a.stride_x_head % xv == 0 &&
                  a.stride_z_token % v == 0 && a.stride_z_head % v == 0 && al16(a.x) && al16(a.z) && al16(a.residual) &&
                  al16(a.weight) && al16(a.y) && al16(a.sum) && al16(a.dy) && al16(a.dsum) && al16(a.dx) && al16(a.dz) &&
                  al16(a.dresidual) && a.group / v <= kMaxVector;
  return ok ? v : 1;
}

struct Shape {
  int ts, iter, threads;  // ts = 0: the CTA is the team
};
// Lanes for n vectors (or scalars) per group.  Few lanes per row keep the
// reductions inside a warp; more than four vectors per lane would spill.
Shape shape_of(int n, bool vec) {
  if (!vec) {
    if (n <= 128) return {32, 4, 256};
    if (n <= 4096) return {0, 4, ((n + 3) / 4 + 31) / 32 * 32};
    return {0, 16, 1024};
  }
  if (n <= 8) return {8, 1, 128};
  if (n <= 16) return {16, 1, 128};
  if (n <= 32) return {32, 1, 128};
  if (n <= 64) return {32, 2, 128};
  if (n <= 128) return {32, 4, 128};
  if (n <= 512) return {0, 2, ((n + 1) / 2 + 31) / 32 * 32};
  if (n <= 1024) return {0, 1, (n + 31) / 32 * 32};
  return {0, 4, 1024};
}
// CTAs per group of the backward: about four per SM over all groups.
int64_t parts_of(const gdn_norm_args& a, const Shape& sh) {
  const int64_t teams = sh.ts ? sh.threads / sh.ts : 1, groups = a.D / a.group;
  return std::max<int64_t>(1, std::min((a.rows + teams - 1) / teams, std::max<int64_t>(1, 592 / groups)));
}

int check(const gdn_norm_args* a, bool bwd) {
  if (!a) return set_last_error(GDN_ERR_INVALID, "null args");
  if (a->rows < 0 || a->heads <= 0 || a->D <= 0 || a->rows % a->heads != 0)
    return set_last_error(GDN_ERR_INVALID, "bad shape rows=%lld heads=%lld D=%lld", (long long)a->rows,
                          (long long)a->heads, (long long)a->D);
  if (a->group <= 0 || a->D % a->group != 0)
    return set_last_error(GDN_ERR_INVALID, "group=%d must divide D=%lld", a->group, (long long)a->D);
  gdn_norm_args v = *a;
  v.x_dtype = a->dtype;  // vectors follow the activations' type
  if (a->group > kMaxScalar && fdtype_ok(a->dtype) && vec_of(v) == 1)
    return set_last_error(GDN_ERR_UNSUPPORTED, "group=%d above %d (or above %d vectors of 16 bytes)", a->group, kMaxScalar,
                          kMaxVector);
  if (a->D / a->group > 65535) return set_last_error(GDN_ERR_UNSUPPORTED, "more than 65535 groups per row");
  if (!fdtype_ok(a->dtype) || !fdtype_ok(a->w_dtype) || !fdtype_ok(a->x_dtype) || !fdtype_ok(a->res_dtype))
    return set_last_error(GDN_ERR_INVALID, "dtypes must be F32, BF16 or F16");
  if (a->x_dtype != a->dtype && !(bwd && a->x_dtype == GDN_F32))
    return set_last_error(GDN_ERR_INVALID, "x must have the activations' dtype (or F32 in the backward)");
  if ((a->residual || a->sum || a->dsum || a->dresidual) && a->res_dtype != a->dtype && a->res_dtype != GDN_F32)
    return set_last_error(GDN_ERR_INVALID, "the residual must have the activations' dtype or F32");
  if (a->activation != GDN_GATE_SILU && a->activation != GDN_GATE_SIGMOID)
    return set_last_error(GDN_ERR_INVALID, "activation must be GDN_GATE_SILU or GDN_GATE_SIGMOID");
  if (a->stride_x_token < 0 || a->stride_x_head < 0 || a->stride_z_token < 0 || a->stride_z_head < 0)
    return set_last_error(GDN_ERR_INVALID, "strides must not be negative");
  return GDN_OK;
}

Params params(const gdn_norm_args& a) {
  Params p{};
  p.x = a.x; p.z = a.z; p.residual = a.residual; p.weight = a.weight; p.y = a.y; p.sum = a.sum;
  p.dy = a.dy; p.dsum = a.dsum; p.dx = a.dx; p.dz = a.dz; p.dresidual = a.dresidual;
  p.partial = static_cast<float*>(a.workspace);
  p.rows = a.rows; p.heads = a.heads; p.D = a.D;
  p.sx_tok = a.stride_x_token; p.sx_head = a.stride_x_head; p.sz_tok = a.stride_z_token; p.sz_head = a.stride_z_head;
  p.group = a.group; p.w_dtype = a.w_dtype; p.res_f32 = a.res_dtype == GDN_F32;
  p.gate_before = a.z && a.gate_before; p.sigmoid_gate = a.activation == GDN_GATE_SIGMOID;
  p.eps = a.eps; p.alpha = a.residual_scale; p.w_off = a.zero_centered ? 1.f : 0.f;
  return p;
}

template <int I>
using Int = std::integral_constant<int, I>;

// Calls f(vectors per thread, lanes per team, largest CTA) of the shape.
template <typename F>
void pick(const Shape& sh, bool vec, F&& f) {
  if (!vec) {
    if (sh.ts == 32) f(Int<4>{}, Int<32>{}, Int<256>{});
    else if (sh.iter == 4) f(Int<4>{}, Int<0>{}, Int<1024>{});
    else f(Int<16>{}, Int<0>{}, Int<1024>{});
    return;
  }
  if (sh.ts == 8) f(Int<1>{}, Int<8>{}, Int<128>{});
  else if (sh.ts == 16) f(Int<1>{}, Int<16>{}, Int<128>{});
  else if (sh.ts == 32 && sh.iter == 1) f(Int<1>{}, Int<32>{}, Int<128>{});
  else if (sh.ts == 32 && sh.iter == 2) f(Int<2>{}, Int<32>{}, Int<128>{});
  else if (sh.ts == 32) f(Int<4>{}, Int<32>{}, Int<128>{});
  else if (sh.iter == 2) f(Int<2>{}, Int<0>{}, Int<256>{});
  else if (sh.iter == 1) f(Int<1>{}, Int<0>{}, Int<1024>{});
  else f(Int<4>{}, Int<0>{}, Int<1024>{});
}

template <typename T, int VEC>
void fwd(const gdn_norm_args& a, const Params& p, cudaStream_t s) {
  const Shape sh = shape_of(a.group / VEC, VEC > 1);
  const int64_t teams = sh.ts ? sh.threads / sh.ts : 1;
  const dim3 grid(static_cast<unsigned>((a.rows + teams - 1) / teams), static_cast<unsigned>(a.D / a.group));
  pick(sh, VEC > 1, [&](auto iter, auto ts, auto most) {
    norm_fwd_kernel<T, VEC, decltype(iter)::value, decltype(ts)::value,
                    decltype(most)::value><<<grid, sh.threads, 0, s>>>(p);
  });
}

template <typename T, typename X, int VEC>
void bwd(const gdn_norm_args& a, const Params& p, cudaStream_t s) {
  const Shape sh = shape_of(a.group / VEC, VEC > 1);
  const int64_t parts = parts_of(a, sh);
  const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>(a.D / a.group));
  const size_t smem = sh.ts ? static_cast<size_t>(sh.threads / sh.ts) * a.group * sizeof(float) : 0;
  pick(sh, VEC > 1, [&](auto iter, auto ts, auto most) {
    norm_bwd_kernel<T, X, VEC, decltype(iter)::value, decltype(ts)::value,
                    decltype(most)::value><<<grid, sh.threads, smem, s>>>(p);
  });
  note_launch();
  norm_dw_kernel<<<static_cast<unsigned>((a.D + 31) / 32), 1024, 0, s>>>(p.partial, parts, a.D, const_cast<void*>(a.dweight),
                                                                       a.w_dtype);
}

template <typename T>
void fwd_t(const gdn_norm_args& a, const Params& p, cudaStream_t s) {
  if (vec_of(a) > 1) fwd<T, 16 / sizeof(T)>(a, p, s);
  else fwd<T, 1>(a, p, s);
}
// Vectors follow the activations' type: eight 16-bit values (and eight fp32
// ones of the residual beside them).
template <typename T, typename X>
void bwd_t(const gdn_norm_args& a, const Params& p, cudaStream_t s) {
  gdn_norm_args b = a;
  b.x_dtype = a.dtype;
  if (vec_of(b) > 1) bwd<T, X, 16 / sizeof(T)>(a, p, s);
  else bwd<T, X, 1>(a, p, s);
}

}  // namespace norm
}  // namespace gdn

using namespace gdn;

extern "C" GDN_API int gdn_norm_fwd(const gdn_norm_args* a, void* stream) {
  const int rc = norm::check(a, false);
  if (rc != GDN_OK) return rc;
  if (a->rows == 0) return GDN_OK;
  if (!a->x || !a->weight || !a->y) return set_last_error(GDN_ERR_INVALID, "x, weight and y must be non-null");
  if ((a->residual != nullptr) != (a->sum != nullptr)) return set_last_error(GDN_ERR_INVALID, "sum goes with residual");
  if (a->rows > 0x7fffffffLL) return set_last_error(GDN_ERR_UNSUPPORTED, "more than 2^31 - 1 rows");
  const norm::Params p = norm::params(*a);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  note_launch();
  if (a->dtype == GDN_F32) norm::fwd_t<float>(*a, p, s);
  else if (a->dtype == GDN_BF16) norm::fwd_t<__nv_bfloat16>(*a, p, s);
  else norm::fwd_t<__half>(*a, p, s);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_last_error(GDN_ERR_CUDA, "gdn_norm_fwd: %s", cudaGetErrorString(e));
  return GDN_OK;
}

// At most 592 CTAs' parts of a row (see parts_of), whatever the alignment.
extern "C" GDN_API size_t gdn_norm_bwd_workspace_size(const gdn_norm_args* a) {
  if (norm::check(a, true)) return 0;
  return static_cast<size_t>(std::max<int64_t>(1, std::min<int64_t>(std::max<int64_t>(a->rows, 1), 592))) * a->D * sizeof(float);
}

extern "C" GDN_API int gdn_norm_bwd(const gdn_norm_args* a, void* stream) {
  const int rc = norm::check(a, true);
  if (rc != GDN_OK) return rc;
  if (!a->weight || !a->dweight || (a->rows > 0 && (!a->x || !a->dy || !a->dx)))
    return set_last_error(GDN_ERR_INVALID, "x, weight, dy, dx and dweight must be non-null");
  if ((a->z != nullptr) != (a->dz != nullptr)) return set_last_error(GDN_ERR_INVALID, "dz goes with z");
  const size_t need = gdn_norm_bwd_workspace_size(a);
  if (!a->workspace || a->workspace_bytes < need)
    return set_last_error(GDN_ERR_WORKSPACE, "workspace of %zu bytes given, %zu needed", a->workspace_bytes, need);
  const norm::Params p = norm::params(*a);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  note_launch();
  const bool xf = a->x_dtype == GDN_F32;
  if (a->dtype == GDN_F32) norm::bwd_t<float, float>(*a, p, s);
  else if (a->dtype == GDN_BF16 && xf) norm::bwd_t<__nv_bfloat16, float>(*a, p, s);
  else if (a->dtype == GDN_BF16) norm::bwd_t<__nv_bfloat16, __nv_bfloat16>(*a, p, s);
  else if (xf) norm::bwd_t<__half, float>(*a, p, s);
  else norm::bwd_t<__half, __half>(*a, p, s);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_last_error(GDN_ERR_CUDA, "gdn_norm_bwd: %s", cudaGetErrorString(e));
  return GDN_OK;
}
