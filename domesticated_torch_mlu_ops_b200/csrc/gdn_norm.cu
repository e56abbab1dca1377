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
// of threads between its reduction and its outputs, one vector per thread: 8,
// 16 or 32 lanes of a warp (several teams per warp share its reductions) up
// to 32 vectors, a whole CTA above.  The backward recomputes rstd (one more
// value in a reduction that it needs anyway) instead of reading a saved one;
// its teams walk the rows of one group with dw in registers, CTAs leave their
// dw in the workspace and a second kernel adds those in order.
//
// Measured: 262144 bf16 rows of 128 with a gate, forward 36 us for 201 MB
// (5.6 TB/s, 85 % of a plain copy's rate), backward 66 + 4 us for 336 MB (4.8
// TB/s); 5001 bf16 rows of 2048 with an fp32 residual, forward 18 us for 123
// MB (the sum stays partly in L2), backward 31 + 4 us for 143 MB.  A few rows
// (64 x 32 of 128): 2.2 us, a launch and one trip to memory.  Rows above 256
// vectors have no look-ahead (larger CTAs, 64 registers) and are slower: 33.5 M
// bf16 values with a gate, forward and backward, 40 and 73 us in rows of 2048,
// 53 and 191 in rows of 2560, 55 and 149 of 4096, 77 and 135 of 5120, 63 and
// 118 of 8192; with an fp32 residual instead 66 and 89, 69 and 250, 69 and 184,
// 86 and 168, 74 and 143.

#include "conv_math.cuh"
#include "gdn_common.cuh"
#include "gdn_internal.h"
#include "packed2.cuh"

#include <algorithm>

namespace gdn {
namespace norm {

using conv::ld_any;
using conv::st_any;

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
  int64_t D;
  int64_t sx_tok, sx_head, sz_tok, sz_head;  // row (t, h) of x and z, in elements
  unsigned rows, heads;
  int group;
  int w_dtype, res_f32, gate_before, sigmoid_gate;
  float eps, alpha, w_off;
};

// act(z) from z and sigmoid(z), and act'(z).
template <int VEC>
__device__ __forceinline__ pk::Vec<VEC> gate(const pk::Vec<VEC>& z, const pk::Vec<VEC>& s, int sigmoid_gate) {
  return sigmoid_gate ? s : pk::mul(z, s);
}
template <int VEC>
__device__ __forceinline__ pk::Vec<VEC> gate_grad(const pk::Vec<VEC>& s, const pk::Vec<VEC>& a, int sigmoid_gate) {
  // silu: s + a (1 - s);  sigmoid: s (1 - s)
  const pk::Vec<VEC> r = pk::fma(s, pk::splat<VEC>(-1.f), pk::splat<VEC>(1.f));
  return sigmoid_gate ? pk::mul(s, r) : pk::fma(a, r, s);
}

template <int VEC>
__device__ __forceinline__ pk::Vec<VEC> ld_weight(const Params& p, int64_t i) {
  pk::Vec<VEC> w;
  if (VEC > 1 && p.w_dtype == GDN_F32) {
    pk::Raw<float, VEC> r;
    pk::load(r, static_cast<const float*>(p.weight) + i);
    w = pk::widen<float, VEC>(r);
  } else if (VEC > 1 && p.w_dtype == GDN_BF16) {
    pk::Raw<__nv_bfloat16, VEC> r;
    pk::load(r, static_cast<const __nv_bfloat16*>(p.weight) + i);
    w = pk::widen<__nv_bfloat16, VEC>(r);
  } else if (VEC > 1) {
    pk::Raw<__half, VEC> r;
    pk::load(r, static_cast<const __half*>(p.weight) + i);
    w = pk::widen<__half, VEC>(r);
  } else {
    pk::set(w, 0, ld_any(p.weight, p.w_dtype, i));
  }
  return pk::add(w, pk::splat<VEC>(p.w_off));
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

// A thread's place in its team, and where its vectors are in a row's group.
// Vectors past the group's end are loaded from its first one and count as 0.
template <int VEC, int ITER, int TS>
struct Team {
  int ts, lane, team, teams, group;
  bool full;  // every vector of every lane lies in the group
  __device__ __forceinline__ explicit Team(int group_) : group(group_) {
    ts = TS ? TS : blockDim.x;
    lane = TS ? threadIdx.x % (TS ? TS : 1) : threadIdx.x;
    team = TS ? threadIdx.x / (TS ? TS : 1) : 0;
    teams = TS ? blockDim.x / (TS ? TS : 1) : 1;
    full = group == ts * ITER * VEC;
  }
  __device__ __forceinline__ int col(int k) const { return (k * ts + lane) * VEC; }
  __device__ __forceinline__ bool in(int k) const { return full || col(k) < group; }
  __device__ __forceinline__ int at(int k) const { return in(k) ? col(k) : 0; }
};

// Rows are counted without sign: up to 2^31 - 1 of them, a step behind the last
// still fits.
__device__ __forceinline__ void row_of(const Params& p, unsigned row, int64_t& x_at, int64_t& z_at) {
  if (p.heads == 1) {
    x_at = row * p.sx_tok;
    z_at = row * p.sz_tok;
  } else {
    const unsigned t = row / p.heads;
    const int64_t h = row - t * p.heads;
    x_at = t * p.sx_tok + h * p.sx_head;
    z_at = t * p.sz_tok + h * p.sz_head;
  }
}

// Rows blockIdx.x * teams + team, + gridDim.x * teams, ...: the next row's
// loads are issued before this one is computed.  R: the residual's type, or
// void without one.
template <typename T, typename R, int VEC, int ITER, int TS, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_fwd_kernel(const Params p) {
  using V = pk::Vec<VEC>;
  constexpr bool kAhead = MAXT <= 256;  // larger CTAs have no registers for the next row
  constexpr bool kRes = !std::is_void<R>::value;
  using RT = typename std::conditional<kRes, R, T>::type;
  __shared__ float buf[2][1][32];
  const Team<VEC, ITER, TS> tm(p.group);
  const int64_t g0 = static_cast<int64_t>(blockIdx.y) * p.group;
  const float inv = 1.f / static_cast<float>(p.group);
  const unsigned step = gridDim.x * tm.teams;
  V w[ITER];
#pragma unroll
  for (int k = 0; k < ITER; ++k) w[k] = ld_weight<VEC>(p, g0 + tm.at(k));
  pk::Raw<T, VEC> rx[ITER], rz[ITER];
  pk::Raw<RT, VEC> rr[ITER];
  auto load = [&](unsigned row) {
    int64_t xa, za;
    row_of(p, min(row, p.rows - 1), xa, za);
    const int64_t at = static_cast<int64_t>(min(row, p.rows - 1)) * p.D + g0;
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      pk::load(rx[k], static_cast<const T*>(p.x) + xa + g0 + tm.at(k));
      if (p.z) pk::load(rz[k], static_cast<const T*>(p.z) + za + g0 + tm.at(k));
      if constexpr (kRes) pk::load_rw(rr[k], static_cast<const RT*>(p.residual) + at + tm.at(k));  // may be the sum
    }
  };
  unsigned row0 = blockIdx.x * tm.teams;
  int par = 0;
  if (kAhead && row0 < p.rows) load(row0 + tm.team);
  // the CTA's teams walk together (shuffles and barriers are for all of them)
  for (; row0 < p.rows; row0 += step) {
    const unsigned row = row0 + tm.team;
    if (!kAhead) load(row);
    V u[ITER], a[ITER];
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      u[k] = pk::widen<T, VEC>(rx[k]);
      if (p.z) a[k] = pk::widen<T, VEC>(rz[k]);
      if constexpr (kRes) u[k] = pk::fma(pk::splat<VEC>(p.alpha), u[k], pk::widen<RT, VEC>(rr[k]));
    }
    if (kAhead && row0 + step < p.rows) load(row + step);
    const bool live = row < p.rows;
    const int64_t at = static_cast<int64_t>(row) * p.D + g0;
    V sq = pk::splat<VEC>(0.f);
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      if constexpr (kRes)
        if (live && tm.in(k)) pk::store<RT, VEC>(static_cast<RT*>(p.sum) + at + tm.col(k), u[k]);
      if (p.z) {
        a[k] = gate(a[k], pk::sigmoid<T>(a[k]), p.sigmoid_gate);
        if (p.gate_before) u[k] = pk::mul(u[k], a[k]);
      }
      if (tm.in(k)) sq = pk::fma(u[k], u[k], sq);
    }
    float ss[1] = {pk::sum(sq)};
    team_sum<TS, 1>(ss, buf[par]);
    par ^= 1;
    const V rstd = pk::splat<VEC>(rsqrtf(fmaf(ss[0], inv, p.eps)));
    if (!live) continue;
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      V y = pk::mul(pk::mul(u[k], rstd), w[k]);
      if (p.z && !p.gate_before) y = pk::mul(y, a[k]);
      if (tm.in(k)) pk::store<T, VEC>(static_cast<T*>(p.y) + at + tm.col(k), y);
    }
  }
}

// X: the type of x (the residual's when the forward summed one).
template <typename T, typename X, int VEC, int ITER, int TS, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_bwd_kernel(const Params p) {
  using V = pk::Vec<VEC>;
  extern __shared__ float dws[];  // [teams][group] when teams > 1
  __shared__ float buf[2][2][32];
  const Team<VEC, ITER, TS> tm(p.group);
  const int64_t g0 = static_cast<int64_t>(blockIdx.y) * p.group;
  const float inv = 1.f / static_cast<float>(p.group);
  const unsigned step = gridDim.x * tm.teams;
  constexpr bool kAhead = MAXT <= 256;  // larger CTAs have no registers for the next row
  V w[ITER], dw[ITER];
#pragma unroll
  for (int k = 0; k < ITER; ++k) {
    w[k] = ld_weight<VEC>(p, g0 + tm.at(k));
    dw[k] = pk::splat<VEC>(0.f);
  }
  pk::Raw<X, VEC> nx[ITER], rs[ITER];
  pk::Raw<T, VEC> nd[ITER], nz[ITER];
  auto load = [&](unsigned row) {
    int64_t xa, za;
    row_of(p, min(row, p.rows - 1), xa, za);
    const int64_t at = static_cast<int64_t>(min(row, p.rows - 1)) * p.D + g0;
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      pk::load(nx[k], static_cast<const X*>(p.x) + xa + g0 + tm.at(k));
      pk::load(nd[k], static_cast<const T*>(p.dy) + at + tm.at(k));
      if (p.z) pk::load(nz[k], static_cast<const T*>(p.z) + za + g0 + tm.at(k));
    }
  };
  unsigned row0 = blockIdx.x * tm.teams;
  int par = 0;
  if (kAhead && row0 < p.rows) load(row0 + tm.team);
  for (; row0 < p.rows; row0 += step) {
    const unsigned row = row0 + tm.team;
    if (!kAhead) load(row);
    const bool live = row < p.rows;
    const int64_t at = static_cast<int64_t>(row) * p.D + g0;
    pk::Raw<X, VEC> rx[ITER];
    pk::Raw<T, VEC> rd[ITER], rz[ITER];
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      rx[k] = nx[k];
      rd[k] = nd[k];
      if (p.z) rz[k] = nz[k];
      if (p.dsum && live) pk::load(rs[k], static_cast<const X*>(p.dsum) + at + tm.at(k));
    }
    if (kAhead && row0 + step < p.rows) load(row + step);
    V s[ITER], squ = pk::splat<VEC>(0.f), sgu = pk::splat<VEC>(0.f);
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      V u = pk::widen<X, VEC>(rx[k]), g = pk::mul(pk::widen<T, VEC>(rd[k]), w[k]);
      if (p.z) {
        const V z = pk::widen<T, VEC>(rz[k]);
        s[k] = pk::sigmoid<T>(z);
        const V a = gate(z, s[k], p.sigmoid_gate);
        if (p.gate_before) u = pk::mul(u, a);
        else g = pk::mul(g, a);
      }
      if (tm.in(k)) {
        squ = pk::fma(u, u, squ);
        sgu = pk::fma(g, u, sgu);
      }
    }
    float sums[2] = {pk::sum(squ), pk::sum(sgu)};
    team_sum<TS, 2>(sums, buf[par]);
    par ^= 1;
    const float rstd = rsqrtf(fmaf(sums[0], inv, p.eps));
    const V rs2 = pk::splat<VEC>(rstd), nc = pk::splat<VEC>(-sums[1] * rstd * inv);  // -mean(dn n)
    if (!live) continue;
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      if (!tm.in(k)) break;
      const V r = pk::widen<X, VEC>(rx[k]), dy = pk::widen<T, VEC>(rd[k]);
      V dr;
      if (!p.z) {
        const V n = pk::mul(r, rs2);
        dw[k] = pk::fma(dy, n, dw[k]);
        dr = pk::mul(rs2, pk::fma(n, nc, pk::mul(dy, w[k])));
      } else {
        const V a = gate(pk::widen<T, VEC>(rz[k]), s[k], p.sigmoid_gate), da = gate_grad(s[k], a, p.sigmoid_gate);
        V dz;
        if (p.gate_before) {
          const V n = pk::mul(pk::mul(r, a), rs2);
          dw[k] = pk::fma(dy, n, dw[k]);
          const V du = pk::mul(rs2, pk::fma(n, nc, pk::mul(dy, w[k])));
          dz = pk::mul(pk::mul(du, r), da);
          dr = pk::mul(du, a);
        } else {
          const V n = pk::mul(r, rs2), g = pk::mul(dy, a), nw = pk::mul(n, w[k]);
          dw[k] = pk::fma(g, n, dw[k]);
          dr = pk::mul(rs2, pk::fma(n, nc, pk::mul(g, w[k])));
          dz = pk::mul(pk::mul(dy, nw), da);
        }
        pk::store<T, VEC>(static_cast<T*>(p.dz) + at + tm.col(k), dz);
      }
      if (p.dsum) dr = pk::add(dr, pk::widen<X, VEC>(rs[k]));
      if (p.dresidual) pk::store<X, VEC>(static_cast<X*>(p.dresidual) + at + tm.col(k), dr);
      pk::store<T, VEC>(static_cast<T*>(p.dx) + at + tm.col(k), pk::mul(dr, pk::splat<VEC>(p.alpha)));
    }
  }
  float* out = p.partial + static_cast<int64_t>(blockIdx.x) * p.D + g0;
  if (TS == 0) {
#pragma unroll
    for (int k = 0; k < ITER; ++k)
      if (tm.in(k))
#pragma unroll
        for (int e = 0; e < VEC; ++e) out[tm.col(k) + e] = pk::get(dw[k], e);
    return;
  }
#pragma unroll
  for (int k = 0; k < ITER; ++k)
    if (tm.in(k))
#pragma unroll
      for (int e = 0; e < VEC; ++e) dws[tm.team * p.group + tm.col(k) + e] = pk::get(dw[k], e);
  __syncthreads();
  for (int i = threadIdx.x; i < p.group; i += blockDim.x) {
    float a = 0.f;
    for (int t = 0; t < tm.teams; ++t) a += dws[t * p.group + i];
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

constexpr int kFwdThreads = 1024, kBwdThreads = 512;  // per SM
constexpr int kMaxScalar = 16 * 1024, kMaxVector = 4 * 1024;  // elements / vectors a CTA can hold

// 16-byte vectors when the group, the strides and every pointer allow them.
int vec_of(const gdn_norm_args& a) {
  const int v = 16 / esize(a.x_dtype);
  const bool ok = a.group % v == 0 && a.D % v == 0 && a.stride_x_token % v == 0 && a.stride_x_head % v == 0 &&
                  a.stride_z_token % v == 0 && a.stride_z_head % v == 0 && al16(a.x) && al16(a.z) && al16(a.residual) &&
                  al16(a.weight) && al16(a.y) && al16(a.sum) && al16(a.dy) && al16(a.dsum) && al16(a.dx) && al16(a.dz) &&
                  al16(a.dresidual) && a.group / v <= kMaxVector;
  return ok ? v : 1;
}

template <int I>
using Int = std::integral_constant<int, I>;

struct Shape {
  int ts, iter, threads;  // ts = 0: the CTA is the team
};

// How a row's group of n vectors (or scalars) is held, as f(vectors per
// thread, lanes per team or 0 for the CTA, largest CTA) and the Shape: one
// vector per thread as far as a CTA reaches.  (Two vectors on half the lanes
// measured the same in the forward, 36 us for 262144 rows of 128 with a gate,
// and cost the backward half its resident threads.)
template <int VEC, typename F>
void pick(int n, F&& f) {
  auto cta = [](int lanes) { return std::max(32, (lanes + 31) / 32 * 32); };
  if constexpr (VEC == 1) {
    if (n <= 128) f(Int<4>{}, Int<32>{}, Int<128>{}, Shape{32, 4, 128});
    else if (n <= 4096) f(Int<4>{}, Int<0>{}, Int<1024>{}, Shape{0, 4, cta((n + 3) / 4)});
    else f(Int<16>{}, Int<0>{}, Int<1024>{}, Shape{0, 16, 1024});
  } else {
    if (n <= 8) f(Int<1>{}, Int<8>{}, Int<128>{}, Shape{8, 1, 128});
    else if (n <= 16) f(Int<1>{}, Int<16>{}, Int<128>{}, Shape{16, 1, 128});
    else if (n <= 32) f(Int<1>{}, Int<32>{}, Int<128>{}, Shape{32, 1, 128});
    else if (n <= 256) f(Int<1>{}, Int<0>{}, Int<256>{}, Shape{0, 1, cta(n)});
    else if (n <= 1024) f(Int<1>{}, Int<0>{}, Int<1024>{}, Shape{0, 1, cta(n)});
    else f(Int<4>{}, Int<0>{}, Int<1024>{}, Shape{0, 4, 1024});
  }
}

// CTAs per group of the backward, over all groups: as many as reside.
int64_t parts_of(const gdn_norm_args& a, const Shape& sh) {
  const int64_t teams = sh.ts ? sh.threads / sh.ts : 1, groups = a.D / a.group;
  const int64_t most = 148 * std::max(1, kBwdThreads / sh.threads);
  return std::max<int64_t>(1, std::min((a.rows + teams - 1) / teams, std::max<int64_t>(1, most / groups)));
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
  if (a->rows > 0x7fffffffLL || a->heads > 0x7fffffffLL)
    return set_last_error(GDN_ERR_UNSUPPORTED, "more than 2^31 - 1 rows");
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
  p.rows = static_cast<unsigned>(a.rows); p.heads = static_cast<unsigned>(a.heads); p.D = a.D;
  p.sx_tok = a.stride_x_token; p.sx_head = a.stride_x_head; p.sz_tok = a.stride_z_token; p.sz_head = a.stride_z_head;
  p.group = a.group; p.w_dtype = a.w_dtype; p.res_f32 = a.res_dtype == GDN_F32;
  p.gate_before = a.z && a.gate_before; p.sigmoid_gate = a.activation == GDN_GATE_SIGMOID;
  p.eps = a.eps; p.alpha = a.residual_scale; p.w_off = a.zero_centered ? 1.f : 0.f;
  if (p.sx_tok == p.heads * p.sx_head && (!a.z || p.sz_tok == p.heads * p.sz_head)) {  // rows in one run
    p.heads = 1;
    p.sx_tok = p.sx_head;
    p.sz_tok = p.sz_head;
  }
  return p;
}

// CTAs per group of the forward: as many as reside, about 1024 threads per SM.
template <typename T, typename R, int VEC>
void fwd(const gdn_norm_args& a, const Params& p, cudaStream_t s) {
  pick<VEC>(a.group / VEC, [&](auto iter, auto ts, auto max_threads, Shape sh) {
    const int64_t teams = sh.ts ? sh.threads / sh.ts : 1, groups = a.D / a.group;
    const int64_t most = std::max<int64_t>(1, 148 * std::max(1, kFwdThreads / sh.threads) / groups);
    const dim3 grid(static_cast<unsigned>(std::min((a.rows + teams - 1) / teams, most)), static_cast<unsigned>(groups));
    norm_fwd_kernel<T, R, VEC, decltype(iter)::value, decltype(ts)::value, decltype(max_threads)::value>
        <<<grid, sh.threads, 0, s>>>(p);
  });
}

template <typename T, typename X, int VEC>
void bwd(const gdn_norm_args& a, const Params& p, cudaStream_t s) {
  pick<VEC>(a.group / VEC, [&](auto iter, auto ts, auto max_threads, Shape sh) {
    const int64_t parts = parts_of(a, sh);
    const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>(a.D / a.group));
    const size_t smem = sh.ts ? static_cast<size_t>(sh.threads / sh.ts) * a.group * sizeof(float) : 0;
    norm_bwd_kernel<T, X, VEC, decltype(iter)::value, decltype(ts)::value, decltype(max_threads)::value>
        <<<grid, sh.threads, smem, s>>>(p);
    note_launch();
    norm_dw_kernel<<<static_cast<unsigned>((a.D + 31) / 32), 1024, 0, s>>>(p.partial, parts, a.D,
                                                                         const_cast<void*>(a.dweight), a.w_dtype);
  });
}

template <typename T>
void fwd_t(const gdn_norm_args& a, const Params& p, cudaStream_t s) {
  const bool vec = vec_of(a) > 1;
  constexpr int kV = 16 / sizeof(T);
  if (!a.residual) vec ? fwd<T, void, kV>(a, p, s) : fwd<T, void, 1>(a, p, s);
  else if (p.res_f32) vec ? fwd<T, float, kV>(a, p, s) : fwd<T, float, 1>(a, p, s);
  else vec ? fwd<T, T, kV>(a, p, s) : fwd<T, T, 1>(a, p, s);
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

// The parts of parts_of at its most (CTAs of 32 threads), whatever the alignment.
extern "C" GDN_API size_t gdn_norm_bwd_workspace_size(const gdn_norm_args* a) {
  if (norm::check(a, true)) return 0;
  return static_cast<size_t>(std::max<int64_t>(1, std::min<int64_t>(std::max<int64_t>(a->rows, 1), 148 * (norm::kBwdThreads / 32)))) * a->D * sizeof(float);
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
