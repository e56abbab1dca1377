// The selective state space scan: the recurrent prompt kernel for every type
// and head size, the kernel that hands states from segment to segment, and
// the C entry points.  The tensor-core prompt kernels are in gdn_scan_tc.cu.
//
// A prompt is cut into segments when there are too few (sequence, head)
// pairs to fill the GPU: the first pass computes the state that each
// segment but the last of a sequence adds, starting from zero, and its log
// decay; scan_pass_kernel turns those into the states the segments start
// from; the second pass computes the outputs (and the last segment's final
// state).  With one segment per sequence the second pass is the only one.

#include "gdn_scan.h"
#include "packed2.cuh"
#include "scan_common.cuh"

#include <algorithm>

namespace gdn {
namespace scan {

constexpr int kTok = 16;  // tokens staged together
constexpr int kUpdWarps = 4;

// Raw inputs of one tile of kTok tokens, on their way to shared memory.
template <typename T, int NB, int NX, bool OUT>
struct RecTile {
  pk::Raw<T, 1> b[NB], c[OUT ? NB : 1], x[NX], z[OUT ? NX : 1];
  float dt;
};

// One CTA per (segment, head, slice of ROWS state rows).  LPR lanes share R
// state rows; each holds SPT of their columns (columns i*4*LPR + 4*lane + e,
// so that the lanes read 16-byte pieces of B and C side by side; R rows use
// what was read, which is what shared memory bounds).  The output sums of R
// rows and four tokens are halved from lane to lane until each lane is left
// with one of them.  Everything in fp32, bound by the fp32 pipes (five packed
// operations per two state elements over both passes; about half their rate):
// 8192 fp16 tokens of 32 heads of 64 x 128 take 216 us (first pass) and 400
// us (319 and 629 with one row per lane group), 1377 fp32 tokens of 6 heads
// of 48 x 40 take 8.3 and 12 us.  A tile's inputs are loaded
// while the tile before it is computed; a tail is padded to four tokens of
// step zero (decay 1, nothing added).
template <typename T, int SPT, int LPR, int R, bool OUT>
__global__ void __launch_bounds__(256, 2) scan_rec_kernel(const ScanParams p) {
  constexpr int SP = SPT * LPR;  // padded state width
  constexpr int ROWS = 256 / LPR * R;
  constexpr int V = 4 * R;  // output sums of four tokens
  static_assert(V <= LPR, "a lane per sum");
  constexpr int NB = kTok * SP / 256, NX = kTok * ROWS / 256;
  __shared__ __align__(16) float sb[kTok][SP], sc[OUT ? kTok : 1][SP], sdt[kTok], sda[kTok], sdecay[kTok];
  __shared__ __align__(16) float sx[kTok][ROWS + 8], sy[OUT ? kTok : 1][ROWS + 8];
  __shared__ int64_t seg_n, seg_t0, seg_t1;
  __shared__ int seg_ok, seg_last;
  const int64_t id = blockIdx.x;
  const int h = blockIdx.y, g = h / (p.H / p.G);
  const int row0 = blockIdx.z * ROWS;
  clear_error(p);
  if (OUT) zero_outside(p, sizeof(T));
  if (threadIdx.x < 32) {
    int64_t n = 0, ls = 0, t0 = 0, t1 = 0;
    bool last = false;
    int64_t chunk0 = 0;
    const bool ok = find_segment(p, id, n, ls, t0, t1, last, chunk0);
    if (threadIdx.x == 0) {
      seg_n = n; seg_t0 = t0; seg_t1 = t1;
      seg_ok = ok; seg_last = last;
    }
  }
  __syncthreads();
  if (!seg_ok || (!OUT && seg_last)) return;
  const int64_t n = seg_n, t0 = seg_t0, t1 = seg_t1;
  const bool last = seg_last;
  const int lane = threadIdx.x % LPR, r = threadIdx.x / LPR * R, row = row0 + r;
  const float A = p.A[h], D = p.D ? p.D[h] : 0.f, bias = p.dt_bias ? p.dt_bias[h] : 0.f;
  const T* bp = static_cast<const T*>(p.b) + static_cast<int64_t>(g) * p.S;
  const T* cp = static_cast<const T*>(p.c) + static_cast<int64_t>(g) * p.S;
  const int64_t col0 = static_cast<int64_t>(h) * p.P + row0;
  RecTile<T, NB, NX, OUT> in;
  auto fetch = [&](int64_t t, int cnt) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int i = threadIdx.x + j * 256, k = i / SP, s = i % SP;
      if (k < cnt && s < p.S) {
        pk::load(in.b[j], bp + (t + k) * p.sb + s);
        if (OUT) pk::load(in.c[j], cp + (t + k) * p.sc + s);
      }
    }
#pragma unroll
    for (int j = 0; j < NX; ++j) {
      const int i = threadIdx.x + j * 256, k = i / ROWS, q = i % ROWS;
      if (k < cnt && row0 + q < p.P) {
        pk::load(in.x[j], static_cast<const T*>(p.x) + (t + k) * p.sx + col0 + q);
        if (OUT && p.z) pk::load(in.z[j], static_cast<const T*>(p.z) + (t + k) * p.sz + col0 + q);
      }
    }
    if (threadIdx.x < cnt) in.dt = ld_any(p.dt, p.dt_dtype, (t + threadIdx.x) * p.sdt + h);
  };
  int cnt = static_cast<int>(min64(kTok, t1 - t0));
  if (t0 < t1) fetch(t0, cnt);
  float2 st[R][SPT / 2];
  const int64_t at_seq = ((n * p.H + h) * p.P + row) * p.S;
  const int64_t at_seg = ((id * p.H + h) * p.P + row) * p.S;
#pragma unroll
  for (int q = 0; q < R; ++q)
#pragma unroll
    for (int i = 0; i < SPT; ++i) {
      const int s = (i / 4) * 4 * LPR + lane * 4 + (i & 3);
      float v = 0.f;
      if (OUT && row + q < p.P && s < p.S) {
        if (p.seg_state) v = p.seg_state[at_seg + q * p.S + s];
        else if (p.init) v = ld_any(p.init, p.init_dtype, at_seq + q * p.S + s);
      }
      if (i & 1) st[q][i / 2].y = v;
      else st[q][i / 2].x = v;
    }
  float logd = 0.f;
  for (int64_t t = t0; t < t1; t += kTok) {
    __syncthreads();  // the tile before this one has been read
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int i = threadIdx.x + j * 256, k = i / SP, s = i % SP;
      const bool there = k < cnt && s < p.S;
      sb[k][s] = there ? pk::widen<T, 1>(in.b[j]).s : 0.f;
      if (OUT) sc[k][s] = there ? pk::widen<T, 1>(in.c[j]).s : 0.f;
    }
#pragma unroll
    for (int j = 0; j < NX; ++j) {
      const int i = threadIdx.x + j * 256, k = i / ROWS, q = i % ROWS;
      sx[k][q] = k < cnt && row0 + q < p.P ? pk::widen<T, 1>(in.x[j]).s : 0.f;
    }
    if (threadIdx.x < kTok) {
      const bool there = threadIdx.x < cnt;
      const float d = there ? step_of(in.dt, bias, p.softplus, p.dt_lo, p.dt_hi) : 0.f, a = there ? d * A : 0.f;
      sdt[threadIdx.x] = d;
      sda[threadIdx.x] = a;
      sdecay[threadIdx.x] = expf(a);
    }
    __syncthreads();
    const int now = cnt;
    pk::Raw<T, 1> z[OUT ? NX : 1];
    if (OUT) {
#pragma unroll
      for (int j = 0; j < NX; ++j) z[j] = in.z[j];
    }
    if (t + kTok < t1) {
      cnt = static_cast<int>(min64(kTok, t1 - t - kTok));
      fetch(t + kTok, cnt);
    }
    for (int k0 = 0; k0 < now; k0 += 4) {
      const float4 dec4 = *reinterpret_cast<const float4*>(&sdecay[k0]), dt4 = *reinterpret_cast<const float4*>(&sdt[k0]);
      float acc[V];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float dec = e == 0 ? dec4.x : e == 1 ? dec4.y : e == 2 ? dec4.z : dec4.w;
        const float dt = e == 0 ? dt4.x : e == 1 ? dt4.y : e == 2 ? dt4.z : dt4.w;
        const float2 dec2 = make_float2(dec, dec);
        float2 u[R], sum[R];
#pragma unroll
        for (int q = 0; q < R; ++q) {
          const float v = dt * sx[k0 + e][r + q];
          u[q] = make_float2(v, v);
          sum[q] = make_float2(0.f, 0.f);
        }
#pragma unroll
        for (int i = 0; i < SPT; i += 4) {
          const int s = i * LPR + lane * 4;
          const float4 b = *reinterpret_cast<const float4*>(&sb[k0 + e][s]);
          float4 c;
          if (OUT) c = *reinterpret_cast<const float4*>(&sc[k0 + e][s]);
#pragma unroll
          for (int q = 0; q < R; ++q) {
            float2 &s0 = st[q][i / 2], &s1 = st[q][i / 2 + 1];
            s0 = __ffma2_rn(dec2, s0, __fmul2_rn(u[q], make_float2(b.x, b.y)));
            s1 = __ffma2_rn(dec2, s1, __fmul2_rn(u[q], make_float2(b.z, b.w)));
            if (OUT) {
              sum[q] = __ffma2_rn(s0, make_float2(c.x, c.y), sum[q]);
              sum[q] = __ffma2_rn(s1, make_float2(c.z, c.w), sum[q]);
            }
          }
        }
#pragma unroll
        for (int q = 0; q < R; ++q) acc[e * R + q] = sum[q].x + sum[q].y;
      }
      if (OUT) {  // lane v of each V ends with sum v: token k0 + v / R, row v % R
#pragma unroll
        for (int m = V / 2; m > 0; m /= 2) {
          const bool up = lane & m;
#pragma unroll
          for (int i = 0; i < m; ++i)
            acc[i] = (up ? acc[i + m] : acc[i]) + __shfl_xor_sync(0xffffffffu, up ? acc[i] : acc[i + m], m);
        }
#pragma unroll
        for (int m = V; m < LPR; m *= 2) acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], m);
        const int k = k0 + lane / R, q = r + lane % R;
        if (lane < V) sy[k][q] = fmaf(D, sx[k][q], acc[0]);
      } else {
        const float4 a = *reinterpret_cast<const float4*>(&sda[k0]);
        logd += (a.x + a.y) + (a.z + a.w);
      }
    }
    if (OUT) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NX; ++j) {
        const int i = threadIdx.x + j * 256, k = i / ROWS, q = i % ROWS;
        if (k >= now || row0 + q >= p.P) continue;
        float v = sy[k][q];
        if (p.z) v *= silu<T>(pk::widen<T, 1>(z[j]).s);
        static_cast<T*>(p.y)[(t + k) * p.H * p.P + col0 + q] = from_f<T>(v);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < R; ++q)
#pragma unroll
    for (int i = 0; i < SPT; ++i) {
      const int s = (i / 4) * 4 * LPR + lane * 4 + (i & 3);
      if (row + q >= p.P || s >= p.S) continue;
      const float v = i & 1 ? st[q][i / 2].y : st[q][i / 2].x;
      if (!OUT) p.seg_state[at_seg + q * p.S + s] = v;
      else if (last && p.final_state) st_any(p.final_state, p.final_dtype, at_seq + q * p.S + s, v);
    }
  if (!OUT && row == 0 && lane == 0) p.seg_decay[id * p.H + h] = logd;
}

// States between segments: for each sequence, head and state element, in
// order of its segments, the state that the segment starts from (in place of
// its first piece's) and h <- exp(log decay) h + state over its pieces.  A
// stream over the pieces' states, eight ahead (one at a time took twice as
// long: 22 segments 11.6 against 5.8 us); VEC elements per thread.
template <int VEC>
__global__ void __launch_bounds__(256) scan_pass_kernel(const ScanParams p) {
  __shared__ int64_t first_sh, count_sh;
  const int64_t n = blockIdx.z;
  const int h = blockIdx.y;
  if (threadIdx.x < 32) {  // the sequence's first segment and their number
    int64_t sum = 0, mine = 0;
    for (int64_t m = threadIdx.x; m <= n; m += 32) {
      int64_t bos, eos;
      seq_bounds(p.cu, p.cu_dtype, m, p.T, bos, eos);
      bos = min64(max(bos, static_cast<int64_t>(0)), p.total);
      eos = min64(max(eos, bos), p.total);
      const int64_t k = max((eos - bos + p.seg - 1) / p.seg, static_cast<int64_t>(1));
      if (m == n) mine = k;
      else sum += k;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      mine += __shfl_xor_sync(0xffffffffu, mine, o);
    }
    if (threadIdx.x == 0) {
      first_sh = sum;
      count_sh = mine;
    }
  }
  __syncthreads();
  const int64_t PS = static_cast<int64_t>(p.P) * p.S;
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * VEC;
  if (i >= PS) return;
  const int64_t first = first_sh, count = min64(count_sh, p.segments - first);
  pk::Vec<VEC> cur;
#pragma unroll
  for (int e = 0; e < VEC; ++e)
    pk::set(cur, e, p.init ? ld_any(p.init, p.init_dtype, (n * p.H + h) * PS + i + e) : 0.f);
  if (count <= 0) return;
  float* st = p.seg_state + (first * p.subs * p.H + h) * PS + i;
  const float* ld = p.seg_decay + first * p.subs * p.H + h;
  const int64_t step = p.H * PS, pieces = (count - 1) * p.subs;  // the last segment adds to nothing here
  constexpr int kAhead = 8;                                      // pieces whose loads are in flight together
  int sub = 0;
  for (int64_t j0 = 0; j0 < pieces; j0 += kAhead) {
    const int now = static_cast<int>(min64(kAhead, pieces - j0));
    pk::Raw<float, VEC> v[kAhead];
    float d[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (j < now) {
        pk::load_rw(v[j], st + j * step);  // overwritten below
        d[j] = ld[j * p.H];
      }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (j < now) {
        if (sub == 0) pk::store<float, VEC>(st + j * step, cur);
        if (++sub == p.subs) sub = 0;
        cur = pk::fma(pk::splat<VEC>(expf(d[j])), cur, pk::widen<float, VEC>(v[j]));
      }
    st += now * step;
    ld += static_cast<int64_t>(now) * p.H;
  }
  pk::store<float, VEC>(st, cur);
}

// ---- single tokens ---------------------------------------------------------
struct UpdateParams {
  const void *x, *dt, *b, *c, *z;
  const float *A, *D, *dt_bias;
  void *state, *y;
  const void* idx;
  int* err;
  int64_t N, slots, s_slot;
  int64_t sx, sdt, sb, sc, sz;
  int H, P, G, S;
  int dt_dtype, idx_dtype, softplus;
  float dt_lo, dt_hi;
};

// The state line of (token, head) is read and written once; nothing else is
// of its size, so HBM bounds the kernel.  LPR lanes hold one row of S (VEC
// columns each, ITER times); a warp moves R rows at a time, all of whose
// loads are in flight together.  256 tokens on fp32 lines of 64 heads x 64 x
// 128 (1.08 GB): 169 us with 32-byte accesses, 98 % of a plain copy's rate.
template <typename T, typename CT, int VEC, int LPR, int ITER, int R>
__global__ void __launch_bounds__(kUpdWarps * 32) scan_update_kernel(const UpdateParams p) {
  constexpr int RW = 32 / LPR;  // rows side by side in a warp
  constexpr int BLK = kUpdWarps * RW * R;
  constexpr bool kWide = VEC * sizeof(CT) == 32;
  const int64_t n = blockIdx.z;
  const int h = blockIdx.y, g = h / (p.H / p.G);
  const int lane = threadIdx.x % LPR, sub = (threadIdx.x & 31) / LPR, warp = threadIdx.x >> 5;
  const int row0 = blockIdx.x * BLK + warp * RW * R + sub;
  const int64_t slot = p.idx ? load_index(p.idx, p.idx_dtype, n) : n;
  T* y = static_cast<T*>(p.y) + (n * p.H + h) * p.P;
  if (slot < 0 || slot >= p.slots) {  // padding, or an index out of the cache: no state, output zero
    if (slot >= p.slots && threadIdx.x == 0 && blockIdx.x == 0 && h == 0)
      record_device_error(p.err, kErrSlotRange, kSiteSlotInitial, static_cast<int>(n), static_cast<int>(slot));
    for (int r = threadIdx.x; r < BLK; r += kUpdWarps * 32)
      if (blockIdx.x * BLK + r < p.P) y[blockIdx.x * BLK + r] = from_f<T>(0.f);
    return;
  }
  CT* st = static_cast<CT*>(p.state) + slot * p.s_slot + static_cast<int64_t>(h) * p.P * p.S;
  pk::Raw<CT, VEC> raw[R][ITER];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      const int row = row0 + r * RW, s = (k * LPR + lane) * VEC;
      const CT* from = st + static_cast<int64_t>(row) * p.S + s;  // replaced below: no load of the read-only kind
      if (row >= p.P || s >= p.S) raw[r][k] = {};
      else if constexpr (kWide) pk::load_rw_wide(raw[r][k], from);
      else pk::load_rw(raw[r][k], from);
    }
  const float dt = step_of(ld_any(p.dt, p.dt_dtype, n * p.sdt + h), p.dt_bias ? p.dt_bias[h] : 0.f, p.softplus,
                           p.dt_lo, p.dt_hi);
  const float decay = expf(dt * p.A[h]), D = p.D ? p.D[h] : 0.f;
  const T* B = static_cast<const T*>(p.b) + n * p.sb + static_cast<int64_t>(g) * p.S;
  const T* C = static_cast<const T*>(p.c) + n * p.sc + static_cast<int64_t>(g) * p.S;
  float bv[ITER][VEC], cv[ITER][VEC];
#pragma unroll
  for (int k = 0; k < ITER; ++k)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int s = (k * LPR + lane) * VEC + e;
      bv[k][e] = s < p.S ? to_f<T>(B[s]) : 0.f;
      cv[k][e] = s < p.S ? to_f<T>(C[s]) : 0.f;
    }
  float out = 0.f;  // row row0 + lane * RW's output, in lane `lane` < R
  const T* x = static_cast<const T*>(p.x) + n * p.sx + static_cast<int64_t>(h) * p.P;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = row0 + r * RW;
    const float xv = row < p.P ? to_f<T>(x[row]) : 0.f, u = dt * xv;
    float acc = 0.f;
#pragma unroll
    for (int k = 0; k < ITER; ++k) {
      const int s = (k * LPR + lane) * VEC;
      pk::Vec<VEC> h = pk::widen<CT, VEC>(raw[r][k]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float v = fmaf(decay, pk::get(h, e), u * bv[k][e]);
        acc = fmaf(v, cv[k][e], acc);
        pk::set(h, e, v);
      }
      if (row < p.P && s < p.S) {
        CT* to = st + static_cast<int64_t>(row) * p.S + s;
        if constexpr (kWide) pk::store_wide(to, reinterpret_cast<const pk::Bits<32>&>(h));
        else pk::store<CT, VEC>(to, h);
      }
    }
    acc = group_sum<LPR>(acc);
    if (lane == r % LPR) {
      float yv = fmaf(D, xv, acc);
      out = yv;
    }
  }
  static_assert(LPR >= R, "a lane per row");
  if (lane < R) {
    const int row = row0 + lane * RW;
    if (row < p.P) {
      if (p.z) out *= silu<T>(to_f<T>(static_cast<const T*>(p.z)[n * p.sz + static_cast<int64_t>(h) * p.P + row]));
      y[row] = from_f<T>(out);
    }
  }
}

// ---- host ------------------------------------------------------------------
bool fdtype_ok(int d) { return d == GDN_F32 || d == GDN_BF16 || d == GDN_F16; }
bool idtype_ok(int d) { return d == GDN_I32 || d == GDN_I64; }

int check(const gdn_scan_args* a) {
  if (!a) return set_last_error(GDN_ERR_INVALID, "null args");
  if (a->B < 0 || a->T < 0 || a->N < 0 || a->H <= 0 || a->P <= 0 || a->G <= 0 || a->S <= 0)
    return set_last_error(GDN_ERR_INVALID, "non-positive dimension (B=%lld T=%lld N=%lld H=%d P=%d G=%d S=%d)",
                          (long long)a->B, (long long)a->T, (long long)a->N, a->H, a->P, a->G, a->S);
  if (a->H % a->G != 0) return set_last_error(GDN_ERR_INVALID, "H=%d is not a multiple of G=%d", a->H, a->G);
  if (a->P > 256 || a->S > 256) return set_last_error(GDN_ERR_UNSUPPORTED, "P=%d, S=%d: both must be <= 256", a->P, a->S);
  if (a->H > 65535 || a->N > 65535) return set_last_error(GDN_ERR_UNSUPPORTED, "H and N must be at most 65535");
  if (a->cu_seqlens) {
    if (!idtype_ok(a->cu_dtype)) return set_last_error(GDN_ERR_INVALID, "cu_seqlens dtype must be I32 or I64");
    if (a->B != 1) return set_last_error(GDN_ERR_INVALID, "cu_seqlens requires B == 1 (got B=%lld)", (long long)a->B);
  } else if (a->N != a->B) {
    return set_last_error(GDN_ERR_INVALID, "without cu_seqlens N must equal B (N=%lld B=%lld)", (long long)a->N,
                          (long long)a->B);
  }
  if (!fdtype_ok(a->dtype) || !fdtype_ok(a->dt_dtype) || !fdtype_ok(a->init_dtype) || !fdtype_ok(a->final_dtype))
    return set_last_error(GDN_ERR_INVALID, "dtypes must be F32, BF16 or F16");
  const int64_t hp = static_cast<int64_t>(a->H) * a->P, gs = static_cast<int64_t>(a->G) * a->S;
  if (a->stride_x < hp || (a->z && a->stride_z < hp) || a->stride_b < gs || a->stride_c < gs || a->stride_dt < a->H)
    return set_last_error(GDN_ERR_INVALID, "token strides must cover a token's packed row");
  if (!(a->dt_min <= a->dt_max)) return set_last_error(GDN_ERR_INVALID, "dt_min must not exceed dt_max");
  return GDN_OK;
}

struct Plan {
  int64_t seg, segments;  // tokens per segment; at most so many segments
  int64_t sub, subs;      // the first pass's pieces of a segment: tokens, number
  bool split;
  size_t scratch_off, state_off, decay_off, bytes;  // the error word comes first
};

// Segment length: enough (segment, head, row slice) CTAs to fill the GPU (one
// per SM on the tensor cores, four of the recurrent kernel), but no segment
// under `least` tokens, below which handing states on costs more than it
// saves: four chunks on the tensor cores, 32 tokens otherwise (1377 tokens of
// 6 heads: 29 us, 31 with 64 tokens; 70 tokens of 24 heads: 27 and 29 us).  Without a device query, so the result depends on
// the shapes alone.
Plan plan(const gdn_scan_args& a) {
  Plan pl{};
  const bool tc = tc_shape(a);
  const int64_t total = a.B * a.T;
  const int64_t slices = tc ? tc_slices(a) : (a.P + 63) / 64;
  const int64_t want = 148 * (tc ? 1 : 4), least = tc ? 512 : 32, unit = tc ? 128 : kTok;
  const int64_t per_token = std::max<int64_t>(1, a.H * slices);
  const int64_t pieces = std::max<int64_t>(1, want / per_token);
  pl.seg = std::max(least, (total + pieces - 1) / pieces);
  pl.seg = (pl.seg + unit - 1) / unit * unit;
  pl.split = a.N > 0 && a.N * per_token < want && total > least;
  if (!pl.split) pl.seg = std::max<int64_t>(128, (total + 127) / 128 * 128);
  // every sequence has at most ceil(len / seg) segments, and at least one
  pl.segments = pl.split ? total / pl.seg + a.N : a.N;
  pl.scratch_off = 256;
  pl.state_off = pl.bytes = 256 + (tc ? (tc_scratch_bytes(a) + 255) / 256 * 256 : 0);
  // The first pass has no chain between its chunks: cut its segments (all but
  // the last of a sequence) further until it fills the GPU too.
  pl.sub = pl.seg;
  if (tc && pl.split) {
    const int64_t cut = std::max<int64_t>(1, want / std::max<int64_t>(1, (pieces - 1) * per_token));
    pl.sub = std::max<int64_t>(128, (pl.seg / cut + 127) / 128 * 128);
  }
  pl.subs = (pl.seg + pl.sub - 1) / pl.sub;
  if (pl.split) {
    const size_t pieces_all = static_cast<size_t>(pl.segments) * pl.subs;
    const size_t states = pieces_all * a.H * a.P * a.S * sizeof(float);
    pl.decay_off = pl.state_off + (states + 255) / 256 * 256;
    pl.bytes = pl.decay_off + pieces_all * a.H * sizeof(float);
  }
  return pl;
}

template <typename T, int SPT, int LPR, int R>
void launch_rec(ScanParams p, const Plan& pl, cudaStream_t s) {
  constexpr int ROWS = 256 / LPR * R;
  const dim3 grid(static_cast<unsigned>(pl.segments), static_cast<unsigned>(p.H),
                  static_cast<unsigned>((p.P + ROWS - 1) / ROWS));
  p.subs = 1;  // this first pass takes whole segments, also in a plan made for the tensor cores
  if (pl.split) {
    note_launch();
    scan_rec_kernel<T, SPT, LPR, R, false><<<grid, 256, 0, s>>>(p);
    launch_pass(p, s);
    p.clear_err = 0;
  }
  note_launch();
  scan_rec_kernel<T, SPT, LPR, R, true><<<grid, 256, 0, s>>>(p);
}

template <typename T>
void launch_t(const ScanParams& p, const Plan& pl, cudaStream_t s) {
  if (p.S <= 16) launch_rec<T, 4, 4, 1>(p, pl, s);
  else if (p.S <= 32) launch_rec<T, 4, 8, 2>(p, pl, s);
  else if (p.S <= 64) launch_rec<T, 4, 16, 4>(p, pl, s);
  else if (p.S <= 128) launch_rec<T, 8, 16, 4>(p, pl, s);
  else launch_rec<T, 16, 16, 2>(p, pl, s);
}

void launch_pass(const ScanParams& p, cudaStream_t s) {
  const int64_t PS = static_cast<int64_t>(p.P) * p.S;
  const int vec = PS % 4 == 0 ? 4 : 1;
  const dim3 grid(static_cast<unsigned>((PS / vec + 255) / 256), static_cast<unsigned>(p.H), static_cast<unsigned>(p.N));
  note_launch();
  if (vec == 4) scan_pass_kernel<4><<<grid, 256, 0, s>>>(p);
  else scan_pass_kernel<1><<<grid, 256, 0, s>>>(p);
}

template <typename T, typename CT, int VEC, int LPR, int ITER, int R>
void launch_upd(const UpdateParams& p, cudaStream_t s) {
  constexpr int BLK = kUpdWarps * (32 / LPR) * R;
  const dim3 grid(static_cast<unsigned>((p.P + BLK - 1) / BLK), static_cast<unsigned>(p.H), static_cast<unsigned>(p.N));
  scan_update_kernel<T, CT, VEC, LPR, ITER, R><<<grid, kUpdWarps * 32, 0, s>>>(p);
}

// Four or five rows per warp, whichever leaves fewer of a CTA's rows idle
// (77 tokens of 40 heads of 80 rows on 16-bit lines: 16 us with five, 20 with
// four, which fills a second CTA's row slots to a quarter).
template <typename T, typename CT, int VEC, int LPR>
void launch_rows(const UpdateParams& p, cudaStream_t s) {
  constexpr int four = kUpdWarps * (32 / LPR) * 4, five = kUpdWarps * (32 / LPR) * 5;
  if ((p.P + five - 1) / five * five < (p.P + four - 1) / four * four) launch_upd<T, CT, VEC, LPR, 1, 5>(p, s);
  else launch_upd<T, CT, VEC, LPR, 1, 4>(p, s);
}

// Lanes per row: S in 32-byte vectors of fp32 lines, or 16-byte ones, where
// the rows allow them, else single columns; four rows per warp and lane in
// flight (256 tokens on fp32 lines of 64 heads x 64 x 128: 169 us; 213 with two
// rows, 192 to 195 with 16-byte vectors and four or eight rows).
template <typename T, typename CT>
void update_t(const UpdateParams& p, cudaStream_t s) {
  constexpr int V = 16 / sizeof(CT);
  auto fits = [&](int v) {
    return p.S % v == 0 && p.s_slot % v == 0 && (reinterpret_cast<uintptr_t>(p.state) & (v * sizeof(CT) - 1)) == 0;
  };
  if constexpr (sizeof(CT) == 4) {
    if (fits(8)) {
      const int n = p.S / 8;
      if (n <= 4) launch_upd<T, CT, 8, 4, 1, 4>(p, s);
      else if (n <= 8) launch_rows<T, CT, 8, 8>(p, s);
      else if (n <= 16) launch_rows<T, CT, 8, 16>(p, s);
      else launch_upd<T, CT, 8, 32, 1, 4>(p, s);
      return;
    }
  }
  if (fits(V)) {
    const int n = p.S / V;
    if (n <= 4) launch_upd<T, CT, V, 4, 1, 4>(p, s);
    else if (n <= 8) launch_rows<T, CT, V, 8>(p, s);
    else if (n <= 16) launch_rows<T, CT, V, 16>(p, s);
    else if (n <= 32) launch_upd<T, CT, V, 32, 1, 4>(p, s);
    else launch_upd<T, CT, V, 32, 2, 4>(p, s);
  } else {
    if (p.S <= 32) launch_upd<T, CT, 1, 32, 1, 8>(p, s);
    else if (p.S <= 128) launch_upd<T, CT, 1, 32, 4, 4>(p, s);
    else launch_upd<T, CT, 1, 32, 8, 4>(p, s);
  }
}

template <typename T>
void update_c(const UpdateParams& p, int state_dtype, cudaStream_t s) {
  if (state_dtype == GDN_F32) update_t<T, float>(p, s);
  else if (state_dtype == GDN_BF16) update_t<T, __nv_bfloat16>(p, s);
  else update_t<T, __half>(p, s);
}

}  // namespace scan
}  // namespace gdn

using namespace gdn;
using namespace gdn::scan;

extern "C" GDN_API size_t gdn_scan_workspace_size(const gdn_scan_args* a) {
  if (check(a)) return 0;
  return plan(*a).bytes;
}

extern "C" GDN_API int gdn_scan_fwd(const gdn_scan_args* a, void* stream) {
  const int rc = check(a);
  if (rc != GDN_OK) return rc;
  const int64_t total = a->B * a->T;
  if (!a->A || (total > 0 && (!a->x || !a->dt || !a->b || !a->c || !a->y)))
    return set_last_error(GDN_ERR_INVALID, "x, dt, A, b, c and y must be non-null");
  const Plan pl = plan(*a);
  if (!a->workspace || a->workspace_bytes < pl.bytes)
    return set_last_error(GDN_ERR_WORKSPACE, "workspace of %zu bytes given, %zu needed", a->workspace_bytes, pl.bytes);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (a->N == 0) {  // no kernel: the error word, and the outputs of tokens without a sequence
    e = cudaMemsetAsync(a->workspace, 0, 4 * sizeof(int32_t), s);
    if (e == cudaSuccess && total > 0)
      e = cudaMemsetAsync(a->y, 0, static_cast<size_t>(total) * a->H * a->P * (a->dtype == GDN_F32 ? 4 : 2), s);
    if (e != cudaSuccess) return set_last_error(GDN_ERR_CUDA, "gdn_scan_fwd: %s", cudaGetErrorString(e));
    return GDN_OK;
  }
  ScanParams p{};
  p.x = a->x; p.dt = a->dt; p.b = a->b; p.c = a->c; p.z = a->z; p.A = a->A; p.D = a->D; p.dt_bias = a->dt_bias;
  p.init = a->initial_state; p.y = a->y; p.final_state = a->final_state; p.cu = a->cu_seqlens;
  if (pl.split) {
    p.seg_state = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + pl.state_off);
    p.seg_decay = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + pl.decay_off);
  }
  p.err = static_cast<int*>(a->workspace);
  p.clear_err = 1;
  p.T = a->T; p.N = a->N; p.total = total; p.seg = pl.seg; p.segments = pl.segments;
  p.sub = pl.sub; p.subs = static_cast<int>(pl.subs);
  p.sx = a->stride_x; p.sdt = a->stride_dt; p.sb = a->stride_b; p.sc = a->stride_c; p.sz = a->stride_z;
  p.H = a->H; p.P = a->P; p.G = a->G; p.S = a->S;
  p.dt_dtype = a->dt_dtype; p.init_dtype = a->init_dtype; p.final_dtype = a->final_dtype; p.cu_dtype = a->cu_dtype;
  p.softplus = a->dt_softplus; p.dt_lo = a->dt_min; p.dt_hi = a->dt_max;
  if (total > 0 && tc_shape(*a) && tc_layout(*a)) e = launch_tc(p, *a, reinterpret_cast<float*>(static_cast<char*>(a->workspace) + pl.scratch_off), s);
  else if (a->dtype == GDN_F32) launch_t<float>(p, pl, s);
  else if (a->dtype == GDN_BF16) launch_t<__nv_bfloat16>(p, pl, s);
  else launch_t<__half>(p, pl, s);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return set_last_error(GDN_ERR_CUDA, "gdn_scan_fwd: %s", cudaGetErrorString(e));
  return GDN_OK;
}

extern "C" GDN_API int gdn_scan_update(const gdn_scan_update_args* a, void* stream) {
  if (!a) return set_last_error(GDN_ERR_INVALID, "null args");
  if (a->N < 0 || a->H <= 0 || a->P <= 0 || a->G <= 0 || a->S <= 0 || a->num_slots < 0)
    return set_last_error(GDN_ERR_INVALID, "non-positive dimension (N=%lld H=%d P=%d G=%d S=%d)", (long long)a->N, a->H,
                          a->P, a->G, a->S);
  if (a->H % a->G != 0) return set_last_error(GDN_ERR_INVALID, "H=%d is not a multiple of G=%d", a->H, a->G);
  if (a->S > 256) return set_last_error(GDN_ERR_UNSUPPORTED, "S=%d must be <= 256", a->S);
  if (a->H > 65535 || a->N > 65535) return set_last_error(GDN_ERR_UNSUPPORTED, "H and N must be at most 65535");
  if (!fdtype_ok(a->dtype) || !fdtype_ok(a->dt_dtype) || !fdtype_ok(a->state_dtype))
    return set_last_error(GDN_ERR_INVALID, "dtypes must be F32, BF16 or F16");
  if (a->ssm_state_indices && !idtype_ok(a->idx_dtype))
    return set_last_error(GDN_ERR_INVALID, "ssm_state_indices dtype must be I32 or I64");
  if (!a->ssm_state_indices && a->num_slots < a->N)
    return set_last_error(GDN_ERR_INVALID, "%lld cache lines for %lld tokens", (long long)a->num_slots, (long long)a->N);
  const int64_t hp = static_cast<int64_t>(a->H) * a->P, gs = static_cast<int64_t>(a->G) * a->S;
  if (a->stride_x < hp || (a->z && a->stride_z < hp) || a->stride_b < gs || a->stride_c < gs || a->stride_dt < a->H ||
      a->stride_slot < hp * a->S)
    return set_last_error(GDN_ERR_INVALID, "strides must cover a token's packed row and a cache line");
  if (!(a->dt_min <= a->dt_max)) return set_last_error(GDN_ERR_INVALID, "dt_min must not exceed dt_max");
  if (a->N == 0) return GDN_OK;
  if (!a->x || !a->dt || !a->A || !a->b || !a->c || !a->state || !a->y)
    return set_last_error(GDN_ERR_INVALID, "x, dt, A, b, c, state and y must be non-null");
  UpdateParams p{};
  p.x = a->x; p.dt = a->dt; p.b = a->b; p.c = a->c; p.z = a->z; p.A = a->A; p.D = a->D; p.dt_bias = a->dt_bias;
  p.state = a->state; p.y = a->y; p.idx = a->ssm_state_indices; p.err = a->err;
  p.N = a->N; p.slots = a->num_slots; p.s_slot = a->stride_slot;
  p.sx = a->stride_x; p.sdt = a->stride_dt; p.sb = a->stride_b; p.sc = a->stride_c; p.sz = a->stride_z;
  p.H = a->H; p.P = a->P; p.G = a->G; p.S = a->S;
  p.dt_dtype = a->dt_dtype; p.idx_dtype = a->idx_dtype; p.softplus = a->dt_softplus;
  p.dt_lo = a->dt_min; p.dt_hi = a->dt_max;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  note_launch();
  if (a->dtype == GDN_F32) update_c<float>(p, a->state_dtype, s);
  else if (a->dtype == GDN_BF16) update_c<__nv_bfloat16>(p, a->state_dtype, s);
  else update_c<__half>(p, a->state_dtype, s);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_last_error(GDN_ERR_CUDA, "gdn_scan_update: %s", cudaGetErrorString(e));
  return GDN_OK;
}
