// Gradient of the causal depthwise conv1d (gdn_causal_conv1d_fwd):
//   pre_t  = bias + sum_i w_i x_{t-W+1+i},  y_t = act(pre_t) + residual_t
//   dpre_t = dy_t act'(pre_t)       silu'(p) = s (1 + p (1 - s)), s = sigmoid(p)
//   dx_s   = sum_k w_{W-1-k} dpre_{s+k}      (s + k inside s's sequence)
//   dw_i   = sum_t dpre_t x_{t-W+1+i},  dbias = sum_t dpre_t
// and the tokens before a sequence start (initial_state) get dx's formula.
//
// pre_t is recomputed from x, so the pass reads x and dy once and writes dx
// once: three streams of the activations, bound by HBM.  As in the forward a
// thread owns one vector of channels and walks a run of tokens; it keeps the
// W-1 previous inputs, the W-1 unfinished dx and the running dw, db in
// registers.  dx_s is complete W-1 tokens later, so a run also reads the W-1
// tokens after its end (the halo: 2 (W-1) tokens per run of at least 64).
// dw and db of a run go to the workspace in fp32 and a second kernel adds
// the runs in their order (4.7 us for 8192 channels): the result does not
// depend on scheduling.

#include "conv_math.cuh"
#include "gdn_common.cuh"
#include "gdn_internal.h"
#include "packed2.cuh"

#include <algorithm>

namespace gdn {
namespace convb {

using namespace conv;

constexpr int kMinRun = 64;  // tokens per run, at least
constexpr int kThreads = 128;
// A thread's vector in bytes, CTAs per SM, and tokens whose loads are in
// flight together at W = 4.  Measured at 8192 tokens x 8192 bf16 channels
// (403 MB): 89 us, 4.5 TB/s, 69 % of a plain copy's rate.  No pipe is full
// (fma 26 %, alu 21 %, special functions 35 %, half of the issue slots) and
// few warps wait for memory: with four warps per scheduler, which the 128
// registers allow, a token's own chain (pre, sigmoid, d, the pending sums) is
// what is left.  Copying the blocks through shared memory (cp.async, 15 tokens
// ahead) took 90 us, 16-byte vectors 91 us, five CTAs per SM 113 us, 4-byte
// vectors 154 us.
constexpr int kVecBytes = 8, kResident = 4, kBlock4 = 6;
constexpr int kMaxW = 16;

struct BwdParams {
  const void* x;
  const void* weight;  // [D, W]
  const void* bias;    // [D] or null
  const void* init;    // [N, D, W] or null
  const void* dy;
  void* dx;
  void* dinit;     // [N, D, W] or null
  float* partial;  // [shares][W + 1][D]: dw taps, then db
  const void* cu;
  int64_t total, D, T, nseq;
  int64_t sx, sdy;  // token strides (elements)
  int64_t nblk, run, shares;
  int W, w_dtype, init_dtype, cu_dtype, act;
};

template <int VEC, int KW, typename T>
struct GradLane {
  using V = pk::Vec<VEC>;
  static constexpr int WM = KW > 0 ? KW : kMaxW;
  static constexpr int WP = WM > 1 ? WM - 1 : 1;
  V w[WM], bias;
  V win[WP];   // win[j] = input at token t - (W-1) + j, j < W-1
  V pend[WP];  // pend[j] = dx so far of token t - (W-1) + j, j < W-1
  V dw[WM], db;
  int w_rt;
  int64_t c;

  __device__ __forceinline__ int width() const { return KW > 0 ? KW : w_rt; }

  __device__ __forceinline__ void init(const BwdParams& p, int64_t c_) {
    w_rt = p.W;
    c = c_;
    const int W = width();
#pragma unroll
    for (int i = 0; i < WM; ++i) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) pk::set(w[i], e, i < W ? ld_any(p.weight, p.w_dtype, (c + e) * W + i) : 0.f);
      dw[i] = pk::splat<VEC>(0.f);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) pk::set(bias, e, p.bias ? ld_any(p.bias, p.w_dtype, c + e) : 0.f);
    db = pk::splat<VEC>(0.f);
  }

  // The window before token t of sequence n = [bos, ...), nothing pending.
  __device__ __forceinline__ void enter(const BwdParams& p, int64_t t, int64_t n, int64_t bos) {
    const int W = width();
#pragma unroll
    for (int j = 0; j < WP; ++j) {
      pend[j] = pk::splat<VEC>(0.f);
      win[j] = pk::splat<VEC>(0.f);
      if (j >= W - 1) continue;
      const int64_t u = t - (W - 1) + j;
      if (u >= bos) {
        pk::Raw<T, VEC> r;
        pk::load(r, static_cast<const T*>(p.x) + u * p.sx + c);
        win[j] = pk::widen<T, VEC>(r);
      } else if (p.init) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          pk::set(win[j], e, ld_any(p.init, p.init_dtype, (n * p.D + c + e) * W + (u - bos) + W));
      }
    }
  }

  // One token: dpre = dy s (1 + pre (1 - s)) with s = sigmoid(pre), its share
  // of dw and db (when `count`), and of the W gradients it reaches; returns
  // the finished one (token t - (W-1)).
  __device__ __forceinline__ V step(const BwdParams& p, const V& xv, const V& dyv, bool count) {
    const int W = width();
    V d = dyv;
    if (p.act == GDN_ACT_SILU) {
      V pre = bias;
#pragma unroll
      for (int j = 0; j < WM - 1; ++j)
        if (j < W - 1) pre = pk::fma(w[j], win[j], pre);
      pre = pk::fma(w[W - 1], xv, pre);
      const V s = pk::sigmoid<T>(pre), one = pk::splat<VEC>(1.f);
      const V r = pk::fma(s, pk::splat<VEC>(-1.f), one);
      d = pk::mul(pk::mul(dyv, s), pk::fma(pre, r, one));
    }
    if (count) {
#pragma unroll
      for (int j = 0; j < WM - 1; ++j)
        if (j < W - 1) dw[j] = pk::fma(d, win[j], dw[j]);
      dw[W - 1] = pk::fma(d, xv, dw[W - 1]);
      db = pk::add(db, d);
    }
    V last = pk::mul(w[W - 1], d), out = last;
    if (W >= 2) {
      out = pk::fma(w[0], d, pend[0]);
#pragma unroll
      for (int j = 0; j + 1 < WM - 1; ++j)
        if (j + 1 < W - 1) {
          pend[j] = pk::fma(w[j + 1], d, pend[j + 1]);
          win[j] = win[j + 1];
        }
      win[W - 2] = xv;
      pend[W - 2] = last;
    }
    return out;
  }
};

// The gradient of token s of sequence n: this run's dx, or (s before the
// sequence start, and the start in this run) a column of dinit.
template <typename T, int VEC>
__device__ __forceinline__ void emit(const BwdParams& p, int64_t s, int64_t t0, int64_t t1, int64_t n, int64_t bos,
                                     int64_t c, int W, const pk::Vec<VEC>& v) {
  if (s >= bos) {
    if (s >= t0 && s < t1) pk::store<T, VEC>(static_cast<T*>(p.dx) + s * p.D + c, v);
  } else if (bos >= t0 && p.dinit) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) st_any(p.dinit, p.init_dtype, (n * p.D + c + e) * W + (s - bos) + W, pk::get(v, e));
  }
}

// U tokens per block, a multiple of W-1 where W is known: the window and the
// pending gradients rotate through their registers and are back in place at a
// block's end, without moves.
template <typename T, int VEC, int KW>
__global__ void __launch_bounds__(kThreads, VEC > 1 && KW > 0 ? kResident : 1) conv_bwd_kernel(const BwdParams p) {
  constexpr int U = KW == 4 ? kBlock4 : 4;
  using V = pk::Vec<VEC>;
  const int64_t cb = blockIdx.x % p.nblk, share = blockIdx.x / p.nblk;
  const int64_t t0 = share * p.run, t1 = min64(p.total, t0 + p.run);
  const int64_t c = (cb * kThreads + threadIdx.x) * VEC;
  if (c >= p.D) return;
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  GradLane<VEC, KW, T> L;
  L.init(p, c);
  const int W = L.width();
  int64_t n, bos, eos;
  if (!p.cu) {
    n = t0 / p.T;
    bos = n * p.T;
    eos = bos + p.T;
  } else {
    int64_t lo = 0, hi = p.nseq;
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) >> 1;
      if (load_index(p.cu, p.cu_dtype, mid) <= t0) lo = mid; else hi = mid;
    }
    n = lo;
    bos = max(load_index(p.cu, p.cu_dtype, n), static_cast<int64_t>(0));
    eos = min64(load_index(p.cu, p.cu_dtype, n + 1), p.total);
  }
  int64_t t = t0;
  while (t < t1) {
    while (t >= eos && n + 1 < p.nseq) {  // next (possibly empty) sequence
      ++n;
      bos = eos;
      eos = p.cu ? min64(load_index(p.cu, p.cu_dtype, n + 1), p.total) : bos + p.T;
    }
    if (t < bos || t >= eos) {  // a token outside every sequence reaches no output
      pk::store<T, VEC>(static_cast<T*>(p.dx) + t * p.D + c, pk::splat<VEC>(0.f));
      ++t;
      continue;
    }
    L.enter(p, t, n, bos);
    const int64_t from = t, stop = min64(eos, t1 + W - 1);
    // a block's loads are issued before the block ahead of it is computed
    pk::Raw<T, VEC> rx[U], rd[U];
    auto load = [&](int64_t at) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int64_t u = min64(at + k, stop - 1);
        pk::load(rx[k], x + u * p.sx + c);
        pk::load(rd[k], dy + u * p.sdy + c);
      }
    };
    load(t);
    while (t < stop) {
      pk::Raw<T, VEC> cx[U], cd[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        cx[k] = rx[k];
        cd[k] = rd[k];
      }
      if (t + U < stop) load(t + U);
      if (t + U <= min64(stop, t1) && t - (W - 1) >= from) {
        // inside the run: every finished gradient is this run's own
        T* out = static_cast<T*>(p.dx) + (t - (W - 1)) * p.D + c;
#pragma unroll
        for (int k = 0; k < U; ++k) {
          pk::store<T, VEC>(out, L.step(p, pk::widen<T, VEC>(cx[k]), pk::widen<T, VEC>(cd[k]), true));
          out += p.D;
        }
        t += U;
      } else {
#pragma unroll
        for (int k = 0; k < U; ++k) {
          if (t < stop) {
            const V out = L.step(p, pk::widen<T, VEC>(cx[k]), pk::widen<T, VEC>(cd[k]), t < t1);
            emit<T, VEC>(p, t - (W - 1), t0, t1, n, bos, c, W, out);
            ++t;
          }
        }
      }
    }
    if (stop == eos) {  // the sequence's last W-1 gradients have no later terms
#pragma unroll
      for (int j = 0; j < GradLane<VEC, KW, T>::WP; ++j)
        if (j < W - 1) emit<T, VEC>(p, eos - (W - 1) + j, t0, t1, n, bos, c, W, L.pend[j]);
    }
  }
  float* out = p.partial + share * (W + 1) * p.D + c;
#pragma unroll
  for (int i = 0; i < GradLane<VEC, KW, T>::WM; ++i)
    if (i < W)
#pragma unroll
      for (int e = 0; e < VEC; ++e) out[i * p.D + e] = pk::get(L.dw[i], e);
#pragma unroll
  for (int e = 0; e < VEC; ++e) out[W * p.D + e] = pk::get(L.db, e);
}

// dw[c][i], db[c] = sum over the runs, in order: eight lanes of runs per
// channel, joined in shared memory.
__global__ void __launch_bounds__(256) conv_bwd_reduce_kernel(const float* partial, int64_t shares, int64_t D, int W,
                                                              void* dw, void* db, int w_dtype) {
  __shared__ float part[8][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  const int i = blockIdx.y;
  float acc = 0.f;
  if (c < D)
    for (int64_t s = row; s < shares; s += 8) acc += partial[(s * (W + 1) + i) * D + c];
  part[row][lane] = acc;
  __syncthreads();
  if (row != 0 || c >= D) return;
#pragma unroll
  for (int r = 1; r < 8; ++r) acc += part[r][lane];
  if (i < W) st_any(dw, w_dtype, c * W + i, acc);
  else if (db) st_any(db, w_dtype, c, acc);
}

bool fdtype_ok(int d) { return d == GDN_F32 || d == GDN_BF16 || d == GDN_F16; }
bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Channels per thread: 8 bytes (4 x 16 bit, or 2 x fp32) when the rows allow
// it, else one.  Wider vectors need more registers for the window, the
// pending gradients and dw than they save in loads.
int vec_of(const gdn_conv1d_bwd_args& a) {
  const int es = a.x_dtype == GDN_F32 ? 4 : 2, v = kVecBytes / es;
  const bool ok = a.D % v == 0 && a.stride_x_token % v == 0 && a.stride_dy_token % v == 0 && aligned(a.x, kVecBytes) &&
                  aligned(a.dy, kVecBytes) && aligned(a.dx, kVecBytes);
  return ok ? v : 1;
}

struct Split {
  int64_t nblk, run, shares;
};
// Equal runs of at least kMinRun tokens, kResident CTAs per SM of 148:
// the same on every device, so the sums' order is too.
Split split_of(int64_t total, int64_t D, int vec) {
  Split s;
  s.nblk = (D + vec * kThreads - 1) / (vec * kThreads);
  s.shares = std::max<int64_t>(1, std::min<int64_t>(148 * kResident / s.nblk, (total + kMinRun - 1) / kMinRun));
  s.run = std::max<int64_t>(1, (total + s.shares - 1) / s.shares);
  s.shares = std::max<int64_t>(1, (total + s.run - 1) / s.run);
  return s;
}

int check(const gdn_conv1d_bwd_args* a) {
  if (!a) return set_last_error(GDN_ERR_INVALID, "null args");
  if (a->B < 0 || a->T < 0 || a->N < 0 || a->D <= 0)
    return set_last_error(GDN_ERR_INVALID, "bad shape B=%lld T=%lld N=%lld D=%lld", (long long)a->B, (long long)a->T,
                          (long long)a->N, (long long)a->D);
  if (a->W < 1 || a->W > kMaxW)
    return set_last_error(GDN_ERR_UNSUPPORTED, "kernel width W=%d outside [1, %d]", a->W, kMaxW);
  if (!fdtype_ok(a->x_dtype) || !fdtype_ok(a->w_dtype) || (a->initial_state && !fdtype_ok(a->state_dtype)))
    return set_last_error(GDN_ERR_INVALID, "x, weight and state dtypes must be F32, BF16 or F16");
  if (a->activation != GDN_ACT_NONE && a->activation != GDN_ACT_SILU)
    return set_last_error(GDN_ERR_INVALID, "activation must be GDN_ACT_NONE or GDN_ACT_SILU");
  if (a->stride_x_token < a->D || a->stride_dy_token < a->D)
    return set_last_error(GDN_ERR_INVALID, "token strides must be at least D=%lld", (long long)a->D);
  if (a->cu_seqlens) {
    if (a->cu_dtype != GDN_I32 && a->cu_dtype != GDN_I64)
      return set_last_error(GDN_ERR_INVALID, "cu_seqlens dtype must be I32 or I64");
    if (a->B != 1) return set_last_error(GDN_ERR_INVALID, "cu_seqlens requires B == 1 (got B=%lld)", (long long)a->B);
    if (a->N < 1) return set_last_error(GDN_ERR_INVALID, "cu_seqlens needs N >= 1 sequences");
  } else if (a->N != a->B) {
    return set_last_error(GDN_ERR_INVALID, "without cu_seqlens N must equal B (N=%lld B=%lld)", (long long)a->N,
                          (long long)a->B);
  }
  if ((a->initial_state != nullptr) != (a->dinitial_state != nullptr))
    return set_last_error(GDN_ERR_INVALID, "dinitial_state goes with initial_state");
  return GDN_OK;
}

template <typename T, int VEC>
void launch_w(const BwdParams& p, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(p.nblk * p.shares);
  note_launch();
  switch (p.W) {
    case 2: conv_bwd_kernel<T, VEC, 2><<<grid, kThreads, 0, s>>>(p); break;
    case 3: conv_bwd_kernel<T, VEC, 3><<<grid, kThreads, 0, s>>>(p); break;
    case 4: conv_bwd_kernel<T, VEC, 4><<<grid, kThreads, 0, s>>>(p); break;
    default: conv_bwd_kernel<T, VEC, 0><<<grid, kThreads, 0, s>>>(p); break;
  }
}

template <typename T>
void launch(const BwdParams& p, int vec, cudaStream_t s) {
  if (vec > 1) launch_w<T, kVecBytes / sizeof(T)>(p, s);
  else launch_w<T, 1>(p, s);
}

}  // namespace convb
}  // namespace gdn

using namespace gdn;

// One size for every alignment (the scalar split has the most channel blocks
// and so the fewest runs), so that the size depends on the shapes alone.
extern "C" GDN_API size_t gdn_causal_conv1d_bwd_workspace_size(const gdn_conv1d_bwd_args* a) {
  if (convb::check(a)) return 0;
  const int es = a->x_dtype == GDN_F32 ? 4 : 2;
  const int64_t total = a->B * a->T;
  const int64_t shares = std::max(convb::split_of(total, a->D, convb::kVecBytes / es).shares, convb::split_of(total, a->D, 1).shares);
  return static_cast<size_t>(shares) * (a->W + 1) * a->D * sizeof(float);
}

extern "C" GDN_API int gdn_causal_conv1d_bwd(const gdn_conv1d_bwd_args* a, void* stream) {
  const int rc = convb::check(a);
  if (rc != GDN_OK) return rc;
  const int64_t total = a->B * a->T;
  if (!a->weight || !a->dweight || (total > 0 && (!a->x || !a->dy || !a->dx)))
    return set_last_error(GDN_ERR_INVALID, "x, weight, dy, dx and dweight must be non-null");
  if ((a->bias != nullptr) != (a->dbias != nullptr)) return set_last_error(GDN_ERR_INVALID, "dbias goes with bias");
  const size_t need = gdn_causal_conv1d_bwd_workspace_size(a);
  if (!a->workspace || a->workspace_bytes < need)
    return set_last_error(GDN_ERR_WORKSPACE, "workspace of %zu bytes given, %zu needed", a->workspace_bytes, need);
  const int vec = convb::vec_of(*a);
  const convb::Split sp = convb::split_of(total, a->D, vec);
  convb::BwdParams p{};
  p.x = a->x; p.weight = a->weight; p.bias = a->bias; p.init = a->initial_state; p.dy = a->dy; p.dx = a->dx;
  p.dinit = a->dinitial_state; p.partial = static_cast<float*>(a->workspace); p.cu = a->cu_seqlens;
  p.total = total; p.D = a->D; p.T = a->T > 0 ? a->T : 1; p.nseq = a->cu_seqlens ? a->N : a->B;
  p.sx = a->stride_x_token; p.sdy = a->stride_dy_token;
  p.nblk = sp.nblk; p.run = sp.run; p.shares = sp.shares;
  p.W = a->W; p.w_dtype = a->w_dtype; p.init_dtype = a->state_dtype; p.cu_dtype = a->cu_dtype; p.act = a->activation;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  // columns that no token reaches (column 0, empty sequences) have gradient 0
  if (p.dinit) e = cudaMemsetAsync(p.dinit, 0, static_cast<size_t>(a->N) * a->D * a->W * (a->state_dtype == GDN_F32 ? 4 : 2), s);
  if (e == cudaSuccess) {
    if (a->x_dtype == GDN_F32) convb::launch<float>(p, vec, s);
    else if (a->x_dtype == GDN_BF16) convb::launch<__nv_bfloat16>(p, vec, s);
    else convb::launch<__half>(p, vec, s);
    note_launch();
    const dim3 grid(static_cast<unsigned>((a->D + 31) / 32), static_cast<unsigned>(a->W + 1));
    convb::conv_bwd_reduce_kernel<<<grid, 256, 0, s>>>(p.partial, p.shares, p.D, p.W, a->dweight, a->dbias, a->w_dtype);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return set_last_error(GDN_ERR_CUDA, "gdn_causal_conv1d_bwd: %s", cudaGetErrorString(e));
  return GDN_OK;
}
