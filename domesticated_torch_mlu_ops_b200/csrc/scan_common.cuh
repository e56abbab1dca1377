// Shared by the selective state space scan's kernels (prompt and single
// token).  Per head h with a scalar decay:
//   dt_t = clamp(softplus(raw_t + bias_h));  a_t = dt_t A_h
//   h_t = exp(a_t) h_{t-1} + dt_t x_t B_t^T          (state [P, S])
//   y_t = (h_t C_t + D_h x_t) silu(z_t)
#pragma once

#include "conv_math.cuh"
#include "gdn_common.cuh"
#include "packed2.cuh"

namespace gdn {
namespace scan {

using conv::ld_any;
using conv::st_any;

// log(1 + e) for 0 <= e <= 1 by the series of the inverse hyperbolic tangent,
// log(1 + e) = 2 (s + s^3/3 + s^5/5 + ...), s = e / (2 + e) <= 1/3: eight
// terms leave a relative error under 2^-26.
__device__ __forceinline__ float log1p_unit(float e) {
  const float s = __fdividef(e, 2.f + e), q = s * s;
  float r = 1.f / 15.f;
  r = fmaf(r, q, 1.f / 13.f);
  r = fmaf(r, q, 1.f / 11.f);
  r = fmaf(r, q, 1.f / 9.f);
  r = fmaf(r, q, 1.f / 7.f);
  r = fmaf(r, q, 1.f / 5.f);
  r = fmaf(r, q, 1.f / 3.f);
  return 2.f * fmaf(s * q, r, s);
}

// The step size: softplus(v) = max(v, 0) + log(1 + exp(-|v|)), exact to a few
// fp32 ulp for every v (the state may be compared in fp32).
__device__ __forceinline__ float step_of(float raw, float bias, int softplus, float lo, float hi) {
  float v = raw + bias;
  if (softplus) v = fmaxf(v, 0.f) + log1p_unit(expf(-fabsf(v)));
  v = v < lo ? lo : v;  // a NaN stays one
  return v > hi ? hi : v;
}

// z / (1 + exp(-z)) for outputs of type T.
template <typename T>
__device__ __forceinline__ float silu(float z) {
  const pk::Vec<1> v{z};
  return z * pk::sigmoid<T>(v).s;
}

struct ScanParams {
  const void *x, *dt, *b, *c, *z;
  const float *A, *D, *dt_bias;
  const void* init;   // [N, H, P, S] or null
  void* y;            // [tokens, H, P]
  void* final_state;  // [N, H, P, S] or null
  const void* cu;
  // segments of seg tokens of each sequence: their states (first the state
  // each adds, then the one it starts from) and log decays
  float* seg_state;  // [segments][H][P][S]
  float* seg_decay;  // [segments][H]
  int* err;          // int32[4] device error word; zeroed by the call's first kernel
  int clear_err;
  int64_t T, N, total, seg, segments;
  int64_t sub;  // the first pass works on pieces of a segment, of sub tokens each
  int subs;     // pieces per segment: seg_state and seg_decay hold that many each

  int64_t sx, sdt, sb, sc, sz;  // token strides
  int H, P, G, S;
  int dt_dtype, init_dtype, final_dtype, cu_dtype, softplus;
  float dt_lo, dt_hi;
};

// Block 0 of the call's first kernel zeroes the error word: it runs long
// before any bounded wait of the call can give up.
__device__ __forceinline__ void clear_error(const ScanParams& p) {
  if (p.clear_err && threadIdx.x < 4 && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) p.err[threadIdx.x] = 0;
}

// Outputs of tokens outside every sequence (before the first, behind the last)
// are zero: by all blocks (x, 0, 0) of a kernel, bytes in all.
__device__ __forceinline__ void zero_outside(const ScanParams& p, int esize) {
  if (!p.cu || blockIdx.y || blockIdx.z) return;
  const int64_t first = min64(max(load_index(p.cu, p.cu_dtype, 0), static_cast<int64_t>(0)), p.total);
  const int64_t end = min64(max(load_index(p.cu, p.cu_dtype, p.N), first), p.total), outside = first + p.total - end;
  if (outside == 0) return;
  char* y = static_cast<char*>(p.y);
  const int64_t row = static_cast<int64_t>(p.H) * p.P * esize;
  const int unit = row % 16 == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0 ? 16 : 2;
  const int64_t head = first * row, gap = (end - first) * row;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * unit; i < outside * row;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x * unit) {
    char* at = y + (i < head ? i : i + gap);
    if (unit == 16) *reinterpret_cast<uint4*>(at) = make_uint4(0u, 0u, 0u, 0u);
    else *reinterpret_cast<uint16_t*>(at) = 0;
  }
}

// Segment `id` of the batch: segment `ls` of sequence n, tokens [t0, t1);
// `last` when it is the sequence's last.  An empty sequence has one empty
// segment.  `chunk0` is the segment's first 128-token chunk, counted over the
// batch (an empty sequence counts as one).  Called by whole warps; false past
// the last segment.
__device__ __forceinline__ bool find_segment(const ScanParams& p, int64_t id, int64_t& n, int64_t& ls, int64_t& t0,
                                             int64_t& t1, bool& last, int64_t& chunk0) {
  const int lane = threadIdx.x & 31;
  int64_t base = 0, base_ch = 0;
  for (int64_t n0 = 0; n0 < p.N; n0 += 32) {
    int64_t bos = 0, eos = 0, mine = 0, mine_ch = 0;
    if (n0 + lane < p.N) {
      seq_bounds(p.cu, p.cu_dtype, n0 + lane, p.T, bos, eos);
      bos = min64(max(bos, static_cast<int64_t>(0)), p.total);
      eos = min64(max(eos, bos), p.total);
      mine = max((eos - bos + p.seg - 1) / p.seg, static_cast<int64_t>(1));
      mine_ch = max((eos - bos + 127) / 128, static_cast<int64_t>(1));
    }
    int64_t incl = mine, incl_ch = mine_ch;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o), w = __shfl_up_sync(0xffffffffu, incl_ch, o);
      if (lane >= o) {
        incl += v;
        incl_ch += w;
      }
    }
    const int64_t total = __shfl_sync(0xffffffffu, incl, 31);
    if (id < base + total) {
      const unsigned hit = __ballot_sync(0xffffffffu, id < base + incl);
      const int src = __ffs(hit) - 1;
      n = n0 + src;
      ls = id - base - __shfl_sync(0xffffffffu, incl - mine, src);
      const int64_t count = __shfl_sync(0xffffffffu, mine, src);
      bos = __shfl_sync(0xffffffffu, bos, src);
      eos = __shfl_sync(0xffffffffu, eos, src);
      t0 = bos + ls * p.seg;
      t1 = min64(eos, t0 + p.seg);
      last = ls + 1 == count;
      chunk0 = base_ch + __shfl_sync(0xffffffffu, incl_ch - mine_ch, src) + (t0 - bos) / 128;
      return true;
    }
    base += total;
    base_ch += __shfl_sync(0xffffffffu, incl_ch, 31);
  }
  return false;
}

}  // namespace scan
}  // namespace gdn
