// Selective scan over prompts on the tensor cores (tcgen05), bf16.
//
// A small kernel first turns the raw steps into what the tiles need per token
// and head: a_i, the log2 decay from the start of the token's 128-token chunk
// to it, and k_i = dt'_i times the decay from it to the end of its block of
// 32 (scan_prep_kernel).
//
// scan_tc_kernel: one CTA per (segment of a sequence, head, 64 columns of P),
// two CTAs per SM.  It walks the segment in chunks of 128 tokens:
//   S  = C B^T                                   [128, 128]
//   Yi = C h                                     [128, 64], h as bf16
//   P_ij = S_ij exp(a_i - a_j) dt'_j  (j <= i)   rounded to bf16 once
//   Ya = P x;   y = exp(a_i) Yi + Ya + D x       in fp32, then the gate
//   dH = B^T (w x),  w_j = exp(a_end - a_j) dt'_j
//   h <- exp(a_end) h + dH                       fp32, in registers
// Four products with fp32 accumulators in TMEM (S and Ya share columns); x, B
// and C come by TMA into 128-byte-swizzled tiles that serve as operands in
// both directions, P replaces C's tile, the second part of w x h's, and y x's
// (from where a TMA store takes it).  The tiles fill half an SM's shared
// memory to the last kilobyte, so there is no second stage; the other CTA
// works while this one waits.
//
// scan_tc_state_kernel, the first pass over split sequences: dH of a whole
// segment in one accumulator, chunks from the last to the first, each
// weighted by the decay to the segment's end.
//
// Rounding.  x, B and C are bf16 already.  P and h are rounded to bf16 as
// operands, as y is rounded to bf16 in the end.  w x is split into bf16 parts
// whose products are summed: two parts (16 bits) where the state only feeds
// y, three (24 bits) where it is returned or handed on, so that a returned
// fp32 state has fp32 precision.
//
// exp(a_i - a_j) = exp(a_i - a_r) (exp(a_r - a_j) dt'_j) with r the end of j's
// block: one exponential per row and block instead of one per element.  Left
// of the diagonal both factors are at most 1.  In the diagonal block the
// first grows as the block decays; above 2^100 that block takes the
// difference itself.  k is summed from the block's end, not as a difference
// of prefix sums, so w keeps its relative precision under fast decays.

#include <cuda.h>

#include "gdn_chunk_tc.cuh"
#include "gdn_scan.h"
#include "scan_common.cuh"

namespace gdn {
namespace scan {

constexpr int kL = 128;             // tokens per chunk
constexpr int kTile = kL * 128;     // 128 rows x 128 bytes (64 bf16 columns)
constexpr int kTcThreads = 256;
constexpr long long kWaitLimit = 2000000000LL;
// The warp that issues copies and products: tokens 0-31 against 64-127, whose
// part of P is all zeros, so it has the least to do while the scores run.
constexpr int kLead = 4;

struct PrepOut {
  float *a, *k, *dt;  // [H][tokens]
};

template <int S_>
struct Smem {
  static constexpr int kB = 0;
  static constexpr int kX = kB + S_ / 64 * kTile;  // x, then y
  static constexpr int kXs = kX + kTile;           // first part of w x (with a third: that, later)
  static constexpr int kH = kXs + kTile;           // h, then the second part of w x
  static constexpr int kC = kH + kTile;            // C, then P
  static constexpr int kCf = kC + 2 * kTile;       // k of the chunk's tokens
  static constexpr int kBar = kCf + kL * 4;        // C and B, x, S and Yi, dH, Ya
  static constexpr int kTmem = kBar + 5 * 8;
  static constexpr int kBytes = kTmem + 8;
  static constexpr int kCols = 256, kYa = 0, kYi = 128, kDH = 192;  // TMEM columns: S (then Ya), Yi, dH
  // two CTAs per SM: 228 KB less 1 KB per CTA
  static_assert(kBytes <= (228 * 1024 - 2 * 1024) / 2, "shared memory");
};

// First pass: B, x, three parts of w x.
template <int S_>
struct StateSmem {
  static constexpr int kB = 0;
  static constexpr int kX = kB + S_ / 64 * kTile;
  static constexpr int kXs = kX + kTile;
  static constexpr int kBar = kXs + 3 * kTile;  // loads, dH
  static constexpr int kTmem = kBar + 2 * 8;
  static constexpr int kBytes = kTmem + 8;
  static constexpr int kCols = 64;
  static constexpr uint32_t kTx = (S_ / 64 + 1) * kTile;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16-byte piece q (of 8) of row r of a swizzled tile.
__device__ __forceinline__ uint4* tile16(uint8_t* tile, int r, int q) {
  return reinterpret_cast<uint4*>(tile + r * 128 + ((q ^ (r & 7)) << 4));
}

__device__ __forceinline__ void unpack8(uint4 u, float2* v) {
  v[0] = conv::unpack2<__nv_bfloat16>(u.x);
  v[1] = conv::unpack2<__nv_bfloat16>(u.y);
  v[2] = conv::unpack2<__nv_bfloat16>(u.z);
  v[3] = conv::unpack2<__nv_bfloat16>(u.w);
}
__device__ __forceinline__ uint4 pack8(const float2* v) {
  return make_uint4(tc::pack_bf16x2(v[0].x, v[0].y), tc::pack_bf16x2(v[1].x, v[1].y),
                    tc::pack_bf16x2(v[2].x, v[2].y), tc::pack_bf16x2(v[3].x, v[3].y));
}
// Eight values as bf16; v keeps what they lost.
__device__ __forceinline__ uint4 take_part(float2* v) {
  const uint4 u = pack8(v);
  float2 h[4];
  unpack8(u, h);
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = __fadd2_rn(v[e], make_float2(-h[e].x, -h[e].y));
  return u;
}

// Steps of one chunk of 128 tokens for 32 heads per block: raw steps in
// through shared memory (rows of heads are what is contiguous), a, k and dt
// out per head with tokens contiguous.  A warp scans a head's 128 tokens,
// four per lane.
__global__ void __launch_bounds__(256) scan_prep_kernel(const ScanParams p, const PrepOut o) {
  __shared__ float raw[kL][33];
  clear_error(p);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h0 = blockIdx.y * 32;
  int64_t n, ls, t0, t1;
  bool last;
  if (!find_segment(p, blockIdx.x, n, ls, t0, t1, last)) return;  // p.seg is the chunk here
  const int len = static_cast<int>(t1 - t0);
  for (int i = warp; i < len; i += 8)
    if (h0 + lane < p.H) raw[i][lane] = ld_any(p.dt, p.dt_dtype, (t0 + i) * p.sdt + h0 + lane);
  __syncthreads();
  for (int hh = warp; hh < 32 && h0 + hh < p.H; hh += 8) {
    const int h = h0 + hh;
    const float A2 = p.A[h] * tc::kLog2e, bias = p.dt_bias ? p.dt_bias[h] : 0.f;
    float d[4], a[4], pre[4], suf[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = lane * 4 + e;
      d[e] = i < len ? step_of(raw[i][hh], bias, p.softplus, p.dt_lo, p.dt_hi) : 0.f;
      a[e] = d[e] * A2;
    }
    pre[0] = a[0];
    suf[3] = 0.f;  // over the later tokens
#pragma unroll
    for (int e = 1; e < 4; ++e) pre[e] = pre[e - 1] + a[e];
#pragma unroll
    for (int e = 2; e >= 0; --e) suf[e] = suf[e + 1] + a[e + 1];
    float up = pre[3], dn = suf[0] + a[0];  // lane totals -> sums over earlier lanes, later lanes of the block
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const float v = __shfl_up_sync(0xffffffffu, up, s);
      if (lane >= s) up += v;
    }
    up = __shfl_up_sync(0xffffffffu, up, 1);
    if (lane == 0) up = 0.f;
#pragma unroll
    for (int s = 1; s < 8; s <<= 1) {  // a block of 32 tokens is 8 lanes
      const float v = __shfl_down_sync(0xffffffffu, dn, s, 8);
      if ((lane & 7) + s < 8) dn += v;
    }
    dn = __shfl_down_sync(0xffffffffu, dn, 1, 8);
    if ((lane & 7) == 7) dn = 0.f;
    const int64_t at = static_cast<int64_t>(h) * p.total + t0 + lane * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane * 4 + e < len) {
        o.a[at + e] = up + pre[e];
        o.k[at + e] = exp2f(suf[e] + dn) * d[e];
        o.dt[at + e] = d[e];
      }
  }
}

// What a thread (token `row` of a chunk) needs of a and k.
struct TokenScalars {
  float a, k;       // its own (0 past the end)
  float end[4];     // a at the end of each block of 32 (of the chunk, past its end)
};
__device__ __forceinline__ TokenScalars load_scalars(const PrepOut& o, int64_t base, int64_t t, int len, int row) {
  TokenScalars s;
  s.a = row < len ? __ldg(o.a + base + t + row) : 0.f;
  s.k = row < len ? __ldg(o.k + base + t + row) : 0.f;
#pragma unroll
  for (int b = 0; b < 4; ++b) s.end[b] = __ldg(o.a + base + t + min(b * 32 + 31, len - 1));
  return s;
}
__device__ __forceinline__ float pick4(const float* v, int q) {
  return q < 2 ? (q == 0 ? v[0] : v[1]) : (q == 2 ? v[2] : v[3]);
}

// What k-step ks of 16 adds to an operand descriptor.
__host__ __device__ constexpr uint64_t k_step(int ks) { return ((ks >> 2) * kTile + (ks & 3) * 32) >> 4; }
__host__ __device__ constexpr uint64_t mn_step(int ks) { return (ks * 2048) >> 4; }

// The swizzled tiles need a 1024-byte-aligned base; there is no static shared
// memory to shift it.
__device__ __forceinline__ bool base_ok(const ScanParams& p, uint32_t sbase) {
  if ((sbase & 1023) == 0) return true;
  if (threadIdx.x == 0) record_device_error(p.err, kErrWaitTimeout, kSiteScanLoad, static_cast<int>(blockIdx.x), -1);
  return false;
}

template <int S_>
__global__ void __launch_bounds__(kTcThreads, 2)
scan_tc_kernel(const ScanParams p, const PrepOut prep, const int slices, const __grid_constant__ CUtensorMap tx,
               const __grid_constant__ CUtensorMap tb, const __grid_constant__ CUtensorMap tcm,
               const __grid_constant__ CUtensorMap ty) {
  using M = Smem<S_>;
  extern __shared__ __align__(1024) uint8_t sm[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + M::kBar);
  uint32_t* tslot = reinterpret_cast<uint32_t*>(sm + M::kTmem);
  const uint32_t sbase = umma::smem_u32(sm);
  const uint32_t bar_cb = umma::smem_u32(bars), bar_x = bar_cb + 8, bar_s = bar_cb + 16, bar_dh = bar_cb + 24,
                 bar_y = bar_cb + 32;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int quad = warp & 3, half = warp >> 2;  // TMEM lane quadrant; column half
  const int row = quad * 32 + lane;             // token of the chunk, or state column s
  // the thread that issues every copy and product (elect.sync picks the same lane each time)
  const bool leader = warp == kLead && umma::elect_one();
  if (!base_ok(p, sbase)) return;
  // Block = segment * units + unit: the CTAs that read the same B and C are
  // adjacent and run together, so those come from L2.
  const int units = p.H * slices;
  const int64_t id = blockIdx.x / units;
  const int unit = static_cast<int>(blockIdx.x - id * units), h = unit / slices, p0 = (unit - h * slices) * 64;
  const int g = h / (p.H / p.G);
  int64_t n = 0, ls = 0, t0 = 0, t1 = 0;
  bool last = false;
  if (!find_segment(p, id, n, ls, t0, t1, last)) return;  // every warp finds the same
  const int nch = static_cast<int>((t1 - t0 + kL - 1) / kL);
  const bool want_state = last && p.final_state;
  const int64_t at_seq = ((n * p.H + h) * p.P + p0 + half * 32) * S_ + row;
  const int64_t at_seg = ((id * p.H + h) * p.P + p0 + half * 32) * S_ + row;
  const float D = p.D ? p.D[h] : 0.f;
  const int64_t prow = static_cast<int64_t>(h) * p.total;
  auto length = [&](int c) { return static_cast<int>(min64(kL, t1 - t0 - static_cast<int64_t>(c) * kL)); };

  // operands of chunk c (one thread)
  auto fetch_c = [&](int c) {
    umma::mbar_arrive_expect_tx(bar_cb, 2 * (S_ / 64) * kTile);
#pragma unroll
    for (int q = 0; q < S_ / 64; ++q)
      umma::tma_load_2d(sm + M::kC + q * kTile, &tcm, g * S_ + q * 64, static_cast<int>(t0) + c * kL, bar_cb);
  };
  auto fetch_b = [&](int c) {
#pragma unroll
    for (int q = 0; q < S_ / 64; ++q)
      umma::tma_load_2d(sm + M::kB + q * kTile, &tb, g * S_ + q * 64, static_cast<int>(t0) + c * kL, bar_cb);
  };
  auto fetch_x = [&](int c) {
    umma::mbar_arrive_expect_tx(bar_x, kTile);
    umma::tma_load_2d(sm + M::kX, &tx, h * p.P + p0, static_cast<int>(t0) + c * kL, bar_x);
  };
  if (leader) {
#pragma unroll
    for (int i = 0; i < 5; ++i) umma::mbar_init(bars + i, 1);
    umma::mbar_fence_init();
    if (nch > 0) {
      fetch_c(0);
      fetch_b(0);
      fetch_x(0);
    }
  }
  if (warp == kLead) {
    umma::tmem_alloc(tslot, M::kCols);
    umma::fence_before_sync();
  }
  TokenScalars sc;
  if (nch > 0) sc = load_scalars(prep, prow, t0, length(0), row);
  // h[s = row][32 columns of P]
  float2 hr[16];
  bool has_h;  // block-uniform: an all-zero state needs no product
  {
    const bool seg = p.seg_state != nullptr, ini = !seg && p.init;
    has_h = seg || ini;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      float v = 0.f;
      if (row < S_) {
        if (seg) v = p.seg_state[at_seg + static_cast<int64_t>(j) * S_];
        else if (ini) v = ld_any(p.init, p.init_dtype, at_seq + static_cast<int64_t>(j) * S_);
      }
      if (j & 1) hr[j / 2].y = v;
      else hr[j / 2].x = v;
    }
  }
  auto store_h = [&]() {
    if (row < S_)
#pragma unroll
      for (int q = 0; q < 4; ++q) *tile16(sm + M::kH, row, half * 4 + q) = pack8(hr + q * 4);
  };
  if (has_h) store_h();
  constexpr uint32_t id_s = umma::idesc_f16(128, 128, true, false, false);
  constexpr uint32_t id_y = umma::idesc_f16(128, 64, true, false, true);
  constexpr uint32_t id_h = umma::idesc_f16(128, 64, true, true, true);
  // operand descriptors: x's and the parts' rows are tokens (K) with 64 columns
  // (N), B is read both ways; a k-step of 16 advances 32 bytes within a
  // K-major atom of 64 columns and 2048 bytes over MN-major rows
  const uint64_t d_c = umma::smem_desc_sw128(sbase + M::kC, 16, 1024), d_bk = umma::smem_desc_sw128(sbase + M::kB, 16, 1024);
  const uint64_t d_bm = umma::smem_desc_sw128(sbase + M::kB, kTile, 1024), d_x = umma::smem_desc_sw128(sbase + M::kX, kTile, 1024);
  const uint64_t d_xs = umma::smem_desc_sw128(sbase + M::kXs, kTile, 1024), d_h = umma::smem_desc_sw128(sbase + M::kH, kTile, 1024);

  bool mine = true;
  int commits_s = 0, commits_dh = 0, commits_y = 0, loads_cb = nch > 0, loads_x = nch > 0;  // so far (leader)
  auto wait = [&](uint32_t bar, uint32_t parity, int site) {
    // one answer per warp: what follows holds warp-wide instructions
    const bool got = __all_sync(0xffffffffu, mine && (umma::mbar_test(bar, parity) || umma::mbar_wait(bar, parity, kWaitLimit)));
    if (mine && !got) record_device_error(p.err, kErrWaitTimeout, site, static_cast<int>(blockIdx.x), tid);
    mine = got;
  };
  uint32_t par_dh = 0, tmem = 0, tl = 0;
  // dH (+)= B^T part.  With S = 64 rows 64-127 of the accumulator are the
  // product of the tile after B: never read.
  auto mma_dh = [&](uint64_t d_part, bool first) {
#pragma unroll
    for (int ks = 0; ks < kL / 16; ++ks)
      umma::mma_f16(tmem + M::kDH, d_bm + mn_step(ks), d_part + mn_step(ks), id_h, !first || ks > 0);
  };
  bool ok = true;
  for (int c = 0; c < nch; ++c) {
    const int64_t tc0 = t0 + static_cast<int64_t>(c) * kL;
    const int len = length(c);
    if (half == 0) reinterpret_cast<float*>(sm + M::kCf)[row] = sc.k;
    const float ai = sc.a, all = sc.end[3], own_end = pick4(sc.end, quad);
    const float wj = sc.k * ex2(all - own_end);
    // ---- S = C B^T, Yi = C h ----
    umma::fence_proxy_async();  // h's tile, and the reads of the tiles that are loaded next
    umma::fence_before_sync();
    if (__syncthreads_or(!mine)) { ok = false; break; }
    umma::fence_after_sync();
    if (c == 0) {
      tmem = __shfl_sync(0xffffffffu, *tslot, 0);
      tl = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    }
    if (warp == kLead) {
      if (c > 0 && umma::elect_one()) {  // y of the last chunk (a whole one) leaves from x's tile
        umma::tma_store_2d(&ty, sm + M::kX, h * p.P + p0, static_cast<int>(tc0 - kL));
        umma::bulk_commit();
      }
      wait(bar_cb, c & 1, kSiteScanLoad);
      if (mine && umma::elect_one()) {
#pragma unroll
        for (int ks = 0; ks < S_ / 16; ++ks) umma::mma_f16(tmem, d_c + k_step(ks), d_bk + k_step(ks), id_s, ks > 0);
        if (has_h)
#pragma unroll
          for (int ks = 0; ks < S_ / 16; ++ks)
            umma::mma_f16(tmem + M::kYi, d_c + k_step(ks), d_h + mn_step(ks), id_y, ks > 0);
        umma::mma_commit(bar_s);
        ++commits_s;
        if (c > 0) {  // x goes where y was
          umma::bulk_wait_read_all();
          fetch_x(c);
          ++loads_x;
        }
      }
      __syncwarp();
    }
    uint4 zr[4];
    const int64_t col = static_cast<int64_t>(h) * p.P + p0 + half * 32;
    if (p.z && row < len) {
      const uint4* zp = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.z) + (tc0 + row) * p.sz + col);
#pragma unroll
      for (int q = 0; q < 4; ++q) zr[q] = __ldg(zp + q);
    }
    // ---- P from the scores ----
    wait(bar_s, c & 1, kSiteScanScores);
    umma::fence_after_sync();
#pragma unroll
    for (int jb = 0; jb < 2; ++jb) {
      const int J = half * 2 + jb;
      uint4 out[4];
      if (J <= quad) {
        float v[32];
        umma::tmem_ld32(tl + J * 32, v);
        const float far = ai - (jb == 0 ? (half == 0 ? sc.end[0] : sc.end[2]) : (half == 0 ? sc.end[1] : sc.end[3]));
        const bool diag = J == quad;
        // far is largest in the block's first row: one answer per warp
        if (!diag || __shfl_sync(0xffffffffu, far, 0) < 100.f) {
          const float f = ex2(far);
          const float2 f2 = make_float2(f, f);
          const float4* cf = reinterpret_cast<const float4*>(sm + M::kCf) + J * 8;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4 k0 = cf[q * 2], k1 = cf[q * 2 + 1];
            float2 w[4] = {make_float2(v[q * 8], v[q * 8 + 1]), make_float2(v[q * 8 + 2], v[q * 8 + 3]),
                           make_float2(v[q * 8 + 4], v[q * 8 + 5]), make_float2(v[q * 8 + 6], v[q * 8 + 7])};
            w[0] = __fmul2_rn(w[0], __fmul2_rn(f2, make_float2(k0.x, k0.y)));
            w[1] = __fmul2_rn(w[1], __fmul2_rn(f2, make_float2(k0.z, k0.w)));
            w[2] = __fmul2_rn(w[2], __fmul2_rn(f2, make_float2(k1.x, k1.y)));
            w[3] = __fmul2_rn(w[3], __fmul2_rn(f2, make_float2(k1.z, k1.w)));
            if (diag)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (q * 8 + e * 2 > lane) w[e].x = 0.f;
                if (q * 8 + e * 2 + 1 > lane) w[e].y = 0.f;
              }
            out[q] = pack8(w);
          }
        } else {
          const float dt = row < len ? __ldg(prep.dt + prow + tc0 + row) : 0.f;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float aj = __shfl_sync(0xffffffffu, ai, j), dj = __shfl_sync(0xffffffffu, dt, j);
            v[j] = j <= lane ? v[j] * (ex2(ai - aj) * dj) : 0.f;
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) out[q] = tc::pack8<__nv_bfloat16>(v + q * 8);
        }
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) out[q] = make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) *tile16(sm + M::kC + half * kTile, row, jb * 4 + q) = out[q];
    }
    // ---- w x in parts ----
    wait(bar_x, c & 1, kSiteScanLoad);
    uint4 low[4];
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint4* xp = tile16(sm + M::kX, row, half * 4 + q);
      uint4 u = *xp;
      if (row >= len) *xp = u = zero;  // another sequence's rows: zero operands, whatever they hold
      float2 v[4];
      unpack8(u, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __fmul2_rn(v[e], make_float2(wj, wj));
      *tile16(sm + M::kXs, row, half * 4 + q) = take_part(v);
      if (want_state) {
        *tile16(sm + M::kH, row, half * 4 + q) = take_part(v);
        low[q] = pack8(v);
      } else {
        *tile16(sm + M::kH, row, half * 4 + q) = pack8(v);
      }
    }
    if (row >= len) {
#pragma unroll
      for (int q = 0; q < S_ / 16; ++q) {
        const int piece = half * (S_ / 16) + q;  // of S_ / 8
        *tile16(sm + M::kB + (piece >> 3) * kTile, row, piece & 7) = zero;
      }
    }
    if (c + 1 < nch) sc = load_scalars(prep, prow, tc0 + kL, length(c + 1), row);
    umma::fence_proxy_async();
    umma::fence_before_sync();
    if (__syncthreads_or(!mine)) { ok = false; break; }
    umma::fence_after_sync();
    if (warp == kLead && umma::elect_one()) {
#pragma unroll
      for (int ks = 0; ks < kL / 16; ++ks)
        umma::mma_f16(tmem + M::kYa, d_c + k_step(ks), d_x + mn_step(ks), id_y, ks > 0);
      umma::mma_commit(bar_y);
      ++commits_y;
      mma_dh(d_xs, true);
      mma_dh(d_h, false);
      umma::mma_commit(bar_dh);
      ++commits_dh;
    }
    __syncwarp();
    // ---- outputs ----
    wait(bar_y, c & 1, kSiteScanOut);
    umma::fence_after_sync();
    if (leader && mine && c + 1 < nch) {
      fetch_c(c + 1);
      ++loads_cb;
    }
    __syncwarp();
    if (mine) {
      const float g1 = ex2(ai);
      const float2 g2 = make_float2(g1, g1), D2 = make_float2(D, D);
      __nv_bfloat16* yp = static_cast<__nv_bfloat16*>(p.y) + (tc0 + row) * p.H * p.P + col;
#pragma unroll
      for (int q2 = 0; q2 < 2; ++q2) {
        float yi[16], ya[16];
        if (has_h) {
          umma::tmem_ld16x2(tl + M::kYi + half * 32 + q2 * 16, tl + M::kYa + half * 32 + q2 * 16, yi, ya);
        } else {
          umma::tmem_ld16(tl + M::kYa + half * 32 + q2 * 16, ya);
#pragma unroll
          for (int e = 0; e < 16; ++e) yi[e] = 0.f;
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint4* xp = tile16(sm + M::kX, row, half * 4 + q2 * 2 + q);
          float2 xv[4], zv[4], o[4];
          unpack8(*xp, xv);
          if (p.z) unpack8(zr[q2 * 2 + q], zv);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = q * 8 + e * 2;
            o[e] = __ffma2_rn(g2, make_float2(yi[i], yi[i + 1]), make_float2(ya[i], ya[i + 1]));
            o[e] = __ffma2_rn(D2, xv[e], o[e]);
            if (p.z) {
              float zz[2] = {zv[e].x, zv[e].y};
              conv::silu_vec<__nv_bfloat16, 2>(zz);
              o[e] = __fmul2_rn(o[e], make_float2(zz[0], zz[1]));
            }
          }
          const uint4 u = pack8(o);
          if (len == kL) *xp = u;
          else if (row < len) *reinterpret_cast<uint4*>(yp + q2 * 16 + q * 8) = u;
        }
      }
    }
    // ---- state ----
    wait(bar_dh, par_dh, kSiteScanState);
    par_dh ^= 1;
    if (want_state) {  // the third part, in the first one's tile
#pragma unroll
      for (int q = 0; q < 4; ++q) *tile16(sm + M::kXs, row, half * 4 + q) = low[q];
      umma::fence_proxy_async();
      umma::fence_before_sync();
      if (__syncthreads_or(!mine)) { ok = false; break; }
      umma::fence_after_sync();
      if (warp == kLead && umma::elect_one()) {
        mma_dh(d_xs, false);
        umma::mma_commit(bar_dh);
        ++commits_dh;
      }
      __syncwarp();
      wait(bar_dh, par_dh, kSiteScanState);
      par_dh ^= 1;
    }
    umma::fence_after_sync();
    if (leader && mine && c + 1 < nch) fetch_b(c + 1);
    __syncwarp();
    const float decay = ex2(all);
    {
      float d[32];
      umma::tmem_ld32(tl + M::kDH + half * 32, d);
#pragma unroll
      for (int j = 0; j < 16; ++j)
        hr[j] = __ffma2_rn(make_float2(decay, decay), hr[j], make_float2(d[j * 2], d[j * 2 + 1]));
    }
    if (c + 1 < nch) store_h();
    has_h = true;
  }
  if (nch > 0) {  // the last chunk's y
    umma::fence_proxy_async();
    umma::fence_before_sync();
    if (ok) ok = !__syncthreads_or(!mine);
    if (ok && leader) {
      if (length(nch - 1) == kL) {
        umma::tma_store_2d(&ty, sm + M::kX, h * p.P + p0, static_cast<int>(t1) - kL);
        umma::bulk_commit();
      }
    }
    __syncwarp();
  }
  if (ok && row < S_ && want_state)
#pragma unroll
    for (int j = 0; j < 32; ++j)
      st_any(p.final_state, p.final_dtype, at_seq + static_cast<int64_t>(j) * S_, j & 1 ? hr[j / 2].y : hr[j / 2].x);
  if (leader) umma::bulk_wait_all();
  if (!ok && leader) {
    // copies and products that this CTA issued may be in flight: wait
    // (bounded) for the last of each before memory is released
    const long long drain = 20000000LL;
    if (loads_cb) umma::mbar_wait(bar_cb, (loads_cb - 1) & 1, drain);
    if (loads_x) umma::mbar_wait(bar_x, (loads_x - 1) & 1, drain);
    if (commits_s) umma::mbar_wait(bar_s, (commits_s - 1) & 1, drain);
    if (commits_y) umma::mbar_wait(bar_y, (commits_y - 1) & 1, drain);
    if (commits_dh) umma::mbar_wait(bar_dh, (commits_dh - 1) & 1, drain);
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  if (warp == kLead) umma::tmem_dealloc(*tslot, M::kCols);
}

template <int S_>
__global__ void __launch_bounds__(kTcThreads, 2)
scan_tc_state_kernel(const ScanParams p, const PrepOut prep, const int slices, const __grid_constant__ CUtensorMap tx,
                     const __grid_constant__ CUtensorMap tb) {
  using M = StateSmem<S_>;
  extern __shared__ __align__(1024) uint8_t sm[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + M::kBar);
  uint32_t* tslot = reinterpret_cast<uint32_t*>(sm + M::kTmem);
  const uint32_t sbase = umma::smem_u32(sm);
  const uint32_t bar_ld = umma::smem_u32(bars), bar_dh = bar_ld + 8;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int quad = warp & 3, half = warp >> 2, row = quad * 32 + lane;
  // the thread that issues every copy and product (elect.sync picks the same lane each time)
  const bool leader = warp == 0 && umma::elect_one();
  if (!base_ok(p, sbase)) return;
  const int units = p.H * slices;
  const int64_t id = blockIdx.x / units;
  const int unit = static_cast<int>(blockIdx.x - id * units), h = unit / slices, p0 = (unit - h * slices) * 64;
  const int g = h / (p.H / p.G);
  int64_t n = 0, ls = 0, t0 = 0, t1 = 0;
  bool last = false;
  if (!find_segment(p, id, n, ls, t0, t1, last) || last) return;
  const int nch = static_cast<int>((t1 - t0) / kL);  // a segment that is not the last is whole chunks
  const int64_t prow = static_cast<int64_t>(h) * p.total;
  auto fetch = [&](int c) {
    const int t = static_cast<int>(t0) + c * kL;
    umma::mbar_arrive_expect_tx(bar_ld, M::kTx);
#pragma unroll
    for (int q = 0; q < S_ / 64; ++q) umma::tma_load_2d(sm + M::kB + q * kTile, &tb, g * S_ + q * 64, t, bar_ld);
    umma::tma_load_2d(sm + M::kX, &tx, h * p.P + p0, t, bar_ld);
  };
  if (leader) {
    umma::mbar_init(bars, 1);
    umma::mbar_init(bars + 1, 1);
    umma::mbar_fence_init();
    fetch(nch - 1);
  }
  if (warp == 0) {
    umma::tmem_alloc(tslot, M::kCols);
    umma::fence_before_sync();
  }
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tslot, 0);
  constexpr uint32_t id_h = umma::idesc_f16(128, 64, true, true, true);
  const uint64_t d_bm = umma::smem_desc_sw128(sbase + M::kB, kTile, 1024), d_xs = umma::smem_desc_sw128(sbase + M::kXs, kTile, 1024);
  bool ok = true, mine = true;
  int loads = 1, commits = 0;
  auto wait = [&](uint32_t bar, uint32_t parity, int site) {
    const bool got = __all_sync(0xffffffffu, mine && (umma::mbar_test(bar, parity) || umma::mbar_wait(bar, parity, kWaitLimit)));
    if (mine && !got) record_device_error(p.err, kErrWaitTimeout, site, static_cast<int>(blockIdx.x), tid);
    mine = got;
  };
  float later = 0.f;  // log2 decay from the chunk's end to the segment's
  TokenScalars sc = load_scalars(prep, prow, t0 + static_cast<int64_t>(nch - 1) * kL, kL, row);
  for (int i = 0; i < nch; ++i) {
    const int c = nch - 1 - i;
    const float wj = sc.k * ex2(sc.end[3] - pick4(sc.end, quad)) * ex2(later);
    later += sc.end[3];
    if (c > 0) sc = load_scalars(prep, prow, t0 + static_cast<int64_t>(c - 1) * kL, kL, row);
    wait(bar_ld, i & 1, kSiteScanLoad);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float2 v[4];
      unpack8(*tile16(sm + M::kX, row, half * 4 + q), v);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __fmul2_rn(v[e], make_float2(wj, wj));
      *tile16(sm + M::kXs, row, half * 4 + q) = take_part(v);
      *tile16(sm + M::kXs + kTile, row, half * 4 + q) = take_part(v);
      *tile16(sm + M::kXs + 2 * kTile, row, half * 4 + q) = pack8(v);
    }
    umma::fence_proxy_async();
    umma::fence_before_sync();
    if (__syncthreads_or(!mine)) { ok = false; break; }
    umma::fence_after_sync();
    if (warp == 0 && umma::elect_one()) {
#pragma unroll
      for (int part = 0; part < 3; ++part)
#pragma unroll
        for (int ks = 0; ks < kL / 16; ++ks)
          umma::mma_f16(tmem, d_bm + mn_step(ks), d_xs + ((part * kTile) >> 4) + mn_step(ks), id_h, i > 0 || part > 0 || ks > 0);
      umma::mma_commit(bar_dh);
      ++commits;
    }
    __syncwarp();
    wait(bar_dh, i & 1, kSiteScanState);
    umma::fence_after_sync();
    if (leader && mine && c > 0) {
      fetch(c - 1);
      ++loads;
    }
    __syncwarp();
  }
  if (ok) ok = !__syncthreads_or(!mine);
  if (ok) {
    float d[32];
    umma::tmem_ld32(tmem + (static_cast<uint32_t>(quad * 32) << 16) + half * 32, d);
    if (row < S_) {
      float* out = p.seg_state + ((id * p.H + h) * p.P + p0 + half * 32) * S_ + row;
#pragma unroll
      for (int j = 0; j < 32; ++j) out[j * S_] = d[j];
    }
    if (tid == 0 && p0 == 0) p.seg_decay[id * p.H + h] = later * 0.6931471805599453f;
  }
  if (!ok && leader) {
    const long long drain = 20000000LL;
    umma::mbar_wait(bar_ld, (loads - 1) & 1, drain);
    if (commits) umma::mbar_wait(bar_dh, (commits - 1) & 1, drain);
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  if (warp == 0) umma::tmem_dealloc(tmem, M::kCols);
}

bool tc_shape(const gdn_scan_args& a) {
  return !a.force_generic && a.dtype == GDN_BF16 && (a.S == 64 || a.S == 128) && a.P % 64 == 0 &&
         a.B * a.T < (int64_t(1) << 31) - kL;
}

int64_t tc_slices(const gdn_scan_args& a) { return a.P / 64; }

// Rows that TMA and 16-byte accesses can read in place.
bool tc_layout(const gdn_scan_args& a) {
  auto al = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  return al(a.x) && al(a.b) && al(a.c) && al(a.z) && al(a.y) && a.stride_x % 8 == 0 && a.stride_b % 8 == 0 &&
         a.stride_c % 8 == 0 && (!a.z || a.stride_z % 8 == 0);
}

// [tokens, columns] bf16 rows with a token stride: boxes of 128 tokens x 64
// columns, 128-byte swizzle; tokens past the end read as zero.
static cudaError_t make_rows_map(CUtensorMap* m, const void* ptr, int64_t cols, int64_t tokens, int64_t stride) {
  auto fn = tc::encode_fn();
  if (!fn) return cudaErrorNotSupported;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(tokens)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * 2};
  const cuuint32_t box[2] = {64, kL}, es[2] = {1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <int S_>
static cudaError_t run_tc(ScanParams p, const gdn_scan_args& a, float* scratch, cudaStream_t s) {
  CUtensorMap tx, tb, tcm, ty;
  cudaError_t e;
  const int64_t total = a.B * a.T, gs = static_cast<int64_t>(a.G) * a.S, hp = static_cast<int64_t>(a.H) * a.P;
  if ((e = make_rows_map(&tx, a.x, hp, total, a.stride_x)) != cudaSuccess) return e;
  if ((e = make_rows_map(&tb, a.b, gs, total, a.stride_b)) != cudaSuccess) return e;
  if ((e = make_rows_map(&tcm, a.c, gs, total, a.stride_c)) != cudaSuccess) return e;
  if ((e = make_rows_map(&ty, a.y, hp, total, hp)) != cudaSuccess) return e;
  const int slices = a.P / 64;
  const PrepOut prep{scratch, scratch + total * a.H, scratch + 2 * total * a.H};
  ScanParams q = p;
  q.seg = kL;
  note_launch();
  scan_prep_kernel<<<dim3(static_cast<unsigned>(total / kL + a.N), static_cast<unsigned>((a.H + 31) / 32)), 256, 0, s>>>(
      q, prep);
  const unsigned grid = static_cast<unsigned>(p.segments * p.H * slices);
  if (p.seg_state) {
    auto kern = scan_tc_state_kernel<S_>;
    if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, StateSmem<S_>::kBytes)) != cudaSuccess)
      return e;
    note_launch();
    kern<<<grid, kTcThreads, StateSmem<S_>::kBytes, s>>>(p, prep, slices, tx, tb);
    launch_pass(p, s);
  }
  auto kern = scan_tc_kernel<S_>;
  if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<S_>::kBytes)) != cudaSuccess)
    return e;
  note_launch();
  kern<<<grid, kTcThreads, Smem<S_>::kBytes, s>>>(p, prep, slices, tx, tb, tcm, ty);
  return cudaGetLastError();
}

size_t tc_scratch_bytes(const gdn_scan_args& a) { return static_cast<size_t>(a.B * a.T) * a.H * 3 * sizeof(float); }

cudaError_t launch_tc(const ScanParams& p, const gdn_scan_args& a, float* scratch, cudaStream_t s) {
  if (p.segments * p.H * (a.P / 64) > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  return a.S == 128 ? run_tc<128>(p, a, scratch, s) : run_tc<64>(p, a, scratch, s);
}

}  // namespace scan
}  // namespace gdn
