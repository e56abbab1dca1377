// Selective scan over prompts on the tensor cores (tcgen05), bf16.
//
// One CTA per (segment of a sequence, head, 64 columns of P), two CTAs per
// SM.  It walks the segment in chunks of 128 tokens; with a_i the log decay
// from the chunk's start to token i and dt' the steps, per chunk:
//   scores  S  = C B^T                           [128, 128]
//   Yi = C h                                     [128, 64], h as bf16
//   P_ij = S_ij exp(a_i - a_j) dt'_j  (j <= i)   rounded to bf16 once
//   Ya = P x;   y = exp(a_i) Yi + Ya + D x       in fp32, then the gate
//   dH = B^T (w x),  w_j = exp(a_end - a_j) dt'_j
//   h <- exp(a_end) h + dH                       fp32, in registers
// Four products with fp32 accumulators in TMEM (S and Ya share columns); x, B
// and C come by TMA into 128-byte-swizzled tiles that serve as operands in
// both directions, P replaces C's tile and the low part of w x replaces h's.
//
// Rounding.  x, B and C are bf16 already.  P and h are rounded to bf16 as
// operands, as y is rounded to bf16 in the end.  w x is split into bf16 parts
// whose products are summed: two parts (16 bits) where the state only feeds
// y, three (24 bits) where it is returned, so that a returned fp32 state has
// fp32 precision.
//
// exp(a_i - a_j) never overflows for decays: blocks of 32 tokens left of the
// diagonal use exp(a_i - a_r) exp(a_r - a_j) with r the end of j's block (both
// factors at most 1; one exponential per row and block instead of one per
// element), the diagonal block the difference itself.  Sums towards the
// chunk's end are taken directly, not as differences of prefix sums: w keeps
// its relative precision under fast decays.
//
// The first pass over split sequences (OUT = false) computes only dH.

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

template <int S_, bool OUT>
struct Smem {
  static constexpr int kB = 0;
  static constexpr int kX = kB + S_ / 64 * kTile;
  static constexpr int kXs = kX + kTile;                      // high part of w x (first pass: all three)
  static constexpr int kH = kXs + (OUT ? 1 : 3) * kTile;      // h, then the middle part of w x
  static constexpr int kC = kH + (OUT ? 1 : 0) * kTile;       // C, then P
  static constexpr int kCf = kC + (OUT ? 2 : 0) * kTile;      // column factors
  static constexpr int kBar = kCf + (OUT ? kL * 4 : 0);       // loads, S and Yi, dH, Ya
  static constexpr int kTmem = kBar + 4 * 8;
  static constexpr int kBytes = kTmem + 8;
  static constexpr int kCols = OUT ? 256 : 64;                // TMEM: S / Ya, Yi, dH
  static constexpr int kDH = OUT ? 192 : 0, kYi = 128, kYa = 0;
  static constexpr uint32_t kTx = (S_ / 64 * (OUT ? 2 : 1) + 1) * kTile;
  // two CTAs per SM: 228 KB less 1 KB per CTA
  static_assert(kBytes <= (228 * 1024 - 2 * 1024) / 2, "shared memory");
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

// Eight values as bf16, and what each lost.
__device__ __forceinline__ uint4 pack_rest(const float* v, float* rest) {
  const uint4 u = tc::pack8<__nv_bfloat16>(v);
  float h[8];
  tc::unpack8<__nv_bfloat16>(u, h);
#pragma unroll
  for (int e = 0; e < 8; ++e) rest[e] = v[e] - h[e];
  return u;
}

template <int S_, bool OUT>
__global__ void __launch_bounds__(kTcThreads, 2)
scan_tc_kernel(const ScanParams p, const int slices, const __grid_constant__ CUtensorMap tx,
               const __grid_constant__ CUtensorMap tb, const __grid_constant__ CUtensorMap tcm) {
  using M = Smem<S_, OUT>;
  extern __shared__ __align__(1024) uint8_t sm[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + M::kBar);
  uint32_t* tslot = reinterpret_cast<uint32_t*>(sm + M::kTmem);
  const uint32_t sbase = umma::smem_u32(sm);
  const uint32_t bar_ld = umma::smem_u32(bars), bar_s = bar_ld + 8, bar_dh = bar_ld + 16, bar_y = bar_ld + 24;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int quad = warp & 3, half = warp >> 2;  // TMEM lane quadrant; column half
  const int row = quad * 32 + lane;             // token of the chunk, or state column s
  clear_error(p);
  if (sbase & 1023) {  // the swizzled tiles need it; there is no static shared memory to shift the base
    if (tid == 0) record_device_error(p.err, kErrWaitTimeout, kSiteScanLoad, static_cast<int>(blockIdx.x), -1);
    return;
  }
  // Block = segment * units + unit: the CTAs that read the same B and C are
  // adjacent and run together, so those come from L2.
  const int units = p.H * slices;
  const int64_t id = blockIdx.x / units;
  const int unit = static_cast<int>(blockIdx.x - id * units), h = unit / slices, p0 = (unit - h * slices) * 64;
  const int g = h / (p.H / p.G);
  int64_t n = 0, ls = 0, t0 = 0, t1 = 0;
  bool last = false;
  if (!find_segment(p, id, n, ls, t0, t1, last)) return;  // every warp finds the same
  if (!OUT && last) return;
  const int nch = static_cast<int>((t1 - t0 + kL - 1) / kL);
  const bool want_state = !OUT || (last && p.final_state);
  const int64_t at_seq = ((n * p.H + h) * p.P + p0 + half * 32) * S_ + row;
  const int64_t at_seg = ((id * p.H + h) * p.P + p0 + half * 32) * S_ + row;
  const float A2 = p.A[h] * tc::kLog2e, bias = p.dt_bias ? p.dt_bias[h] : 0.f, D = p.D ? p.D[h] : 0.f;

  // operands of chunk c (one thread)
  auto fetch = [&](int c) {
    const int t = static_cast<int>(t0) + c * kL;
    umma::mbar_arrive_expect_tx(bar_ld, M::kTx);
#pragma unroll
    for (int q = 0; q < S_ / 64; ++q) {
      if (OUT) umma::tma_load_2d(sm + M::kC + q * kTile, &tcm, g * S_ + q * 64, t, bar_ld);
      umma::tma_load_2d(sm + M::kB + q * kTile, &tb, g * S_ + q * 64, t, bar_ld);
    }
    umma::tma_load_2d(sm + M::kX, &tx, h * p.P + p0, t, bar_ld);
  };
  // raw steps of chunk c: token b * 32 + lane in raw[b]
  float raw[4];
  auto fetch_dt = [&](int c) {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int64_t t = t0 + static_cast<int64_t>(c) * kL + b * 32 + lane;
      raw[b] = t < t1 ? ld_any(p.dt, p.dt_dtype, t * p.sdt + h) : 0.f;
    }
  };
  if (nch > 0) fetch_dt(0);
  if (tid == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) umma::mbar_init(bars + i, 1);
    umma::mbar_fence_init();
    if (nch > 0) fetch(0);
  }
  if (warp == 0) {
    umma::tmem_alloc(tslot, M::kCols);
    umma::fence_before_sync();
  }
  // h[s = row][32 columns of P]
  float hr[32];
  bool has_h = false;  // block-uniform: an all-zero state needs no product
  {
    const bool seg = OUT && p.seg_state, ini = OUT && !p.seg_state && p.init;
    has_h = seg || ini;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      hr[j] = 0.f;
      if (row < S_) {
        if (seg) hr[j] = p.seg_state[at_seg + static_cast<int64_t>(j) * S_];
        else if (ini) hr[j] = ld_any(p.init, p.init_dtype, at_seq + static_cast<int64_t>(j) * S_);
      }
    }
  }
  auto store_h = [&]() {
    if (row < S_)
#pragma unroll
      for (int q = 0; q < 4; ++q) *tile16(sm + M::kH, row, half * 4 + q) = tc::pack8<__nv_bfloat16>(hr + q * 8);
  };
  if (OUT && has_h) store_h();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = *tslot;
  const uint32_t tl = tmem + (static_cast<uint32_t>(quad * 32) << 16);
  constexpr uint32_t id_s = umma::idesc_f16(128, 128, true, false, false);
  constexpr uint32_t id_y = umma::idesc_f16(128, 64, true, false, true);
  constexpr uint32_t id_h = umma::idesc_f16(128, 64, true, true, true);
  auto kmajor = [&](int off, int ks) {
    return umma::smem_desc_sw128(sbase + off + (ks >> 2) * kTile + (ks & 3) * 32, 16, 1024);
  };
  auto mnmajor = [&](int off, int ks) { return umma::smem_desc_sw128(sbase + off + ks * 2048, kTile, 1024); };
  // dH (+)= B^T part.  With S = 64 rows 64-127 of the accumulator are the
  // product of the tile after B: never read.
  auto mma_dh = [&](int part_off, bool first) {
#pragma unroll
    for (int ks = 0; ks < kL / 16; ++ks)
      umma::mma_f16(tmem + M::kDH, mnmajor(M::kB, ks), mnmajor(part_off, ks), id_h, !first || ks > 0);
  };

  bool ok = true, mine = true;
  uint32_t par_dh = 0;
  int commits_s = 0, commits_dh = 0, commits_y = 0, loads = nch > 0 ? 1 : 0;  // issued so far (thread 0)
  auto wait = [&](uint32_t bar, uint32_t parity, int site) {
    // one answer per warp: what follows holds warp-wide instructions
    const bool got = __all_sync(0xffffffffu, mine && umma::mbar_wait(bar, parity, kWaitLimit));
    if (mine && !got) record_device_error(p.err, kErrWaitTimeout, site, static_cast<int>(blockIdx.x), tid);
    mine = got;
  };
  float logd = 0.f;
  for (int c = 0; c < nch; ++c) {
    const int64_t tc0 = t0 + static_cast<int64_t>(c) * kL;
    const int len = static_cast<int>(min64(kL, t1 - tc0));
    // ---- steps and their sums (every warp, for all 128 tokens) ----
    float tot[4], pin = 0.f, suf = 0.f, dt = 0.f, before = 0.f, after = 0.f;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const float d = b * 32 + lane < len ? step_of(raw[b], bias, p.softplus, p.dt_lo, p.dt_hi) : 0.f;
      const float a = d * A2;
      float up = a;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float v = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += v;
      }
      tot[b] = __shfl_sync(0xffffffffu, up, 31);
      if (b == quad) {
        float dn = __shfl_down_sync(0xffffffffu, a, 1);  // sum over the later tokens of the block
        if (lane == 31) dn = 0.f;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const float v = __shfl_down_sync(0xffffffffu, dn, o);
          if (lane + o < 32) dn += v;
        }
        pin = up;
        suf = dn;
        dt = d;
      }
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (b < quad) before += tot[b];
      if (b > quad) after += tot[b];
    }
    const float all = tot[0] + tot[1] + tot[2] + tot[3];
    logd += all;
    if (c + 1 < nch) fetch_dt(c + 1);
    if (OUT && half == 0) reinterpret_cast<float*>(sm + M::kCf)[row] = ex2(suf) * dt;
    const float wj = ex2(suf + after) * dt;

    // ---- w x in parts ----
    wait(bar_ld, c & 1, kSiteScanLoad);
    uint4 mid[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float v[8], rest[8], low[8];
      tc::unpack8<__nv_bfloat16>(*tile16(sm + M::kX, row, half * 4 + q), v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = row < len ? v[e] * wj : 0.f;
      *tile16(sm + M::kXs, row, half * 4 + q) = pack_rest(v, rest);
      mid[q] = pack_rest(rest, low);
      if (!OUT) {
        *tile16(sm + M::kXs + kTile, row, half * 4 + q) = mid[q];
        *tile16(sm + M::kXs + 2 * kTile, row, half * 4 + q) = tc::pack8<__nv_bfloat16>(low);
      }
    }
    if (row >= len) {  // another sequence's rows: zero operands, whatever they hold
      const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int q = 0; q < 4; ++q) *tile16(sm + M::kX, row, half * 4 + q) = zero;
#pragma unroll
      for (int q = 0; q < S_ / 16; ++q) {
        const int col = half * (S_ / 16) + q;  // of S_ / 8 pieces
        *tile16(sm + M::kB + (col >> 3) * kTile, row, col & 7) = zero;
      }
    }
    umma::fence_proxy_async();
    umma::fence_before_sync();
    if (__syncthreads_or(!mine)) { ok = false; break; }
    umma::fence_after_sync();
    if (tid == 0) {
      if (OUT) {
#pragma unroll
        for (int ks = 0; ks < S_ / 16; ++ks) umma::mma_f16(tmem, kmajor(M::kC, ks), kmajor(M::kB, ks), id_s, ks > 0);
        if (has_h)
#pragma unroll
          for (int ks = 0; ks < S_ / 16; ++ks)
            umma::mma_f16(tmem + M::kYi, kmajor(M::kC, ks), mnmajor(M::kH, ks), id_y, ks > 0);
        umma::mma_commit(bar_s);
        ++commits_s;
        mma_dh(M::kXs, true);
      } else {
        mma_dh(M::kXs, true);
        mma_dh(M::kXs + kTile, false);
        mma_dh(M::kXs + 2 * kTile, false);
        umma::mma_commit(bar_dh);
        ++commits_dh;
      }
    }
    __syncwarp();
    if constexpr (OUT) {
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
        float v[32];
        if (J <= quad) {
          umma::tmem_ld32(tl + J * 32, v);
          if (J < quad) {
            float f = pin;
#pragma unroll
            for (int b = 1; b < 3; ++b)
              if (b > J && b < quad) f += tot[b];
            f = ex2(f);
            const float4* cf = reinterpret_cast<const float4*>(sm + M::kCf) + J * 8;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const float4 k = cf[q];
              v[q * 4] *= f * k.x;
              v[q * 4 + 1] *= f * k.y;
              v[q * 4 + 2] *= f * k.z;
              v[q * 4 + 3] *= f * k.w;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const float aj = __shfl_sync(0xffffffffu, pin, j), dj = __shfl_sync(0xffffffffu, dt, j);
              v[j] = j <= lane ? v[j] * (ex2(pin - aj) * dj) : 0.f;
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0.f;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *tile16(sm + M::kC + half * kTile, row, jb * 4 + q) = tc::pack8<__nv_bfloat16>(v + q * 8);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) *tile16(sm + M::kH, row, half * 4 + q) = mid[q];
      umma::fence_proxy_async();
      umma::fence_before_sync();
      if (__syncthreads_or(!mine)) { ok = false; break; }
      umma::fence_after_sync();
      if (tid == 0) {
#pragma unroll
        for (int ks = 0; ks < kL / 16; ++ks)
          umma::mma_f16(tmem + M::kYa, kmajor(M::kC, ks), mnmajor(M::kX, ks), id_y, ks > 0);
        umma::mma_commit(bar_y);
        ++commits_y;
        mma_dh(M::kH, false);
        umma::mma_commit(bar_dh);
        ++commits_dh;
      }
      __syncwarp();
      // ---- outputs ----
      wait(bar_y, c & 1, kSiteScanOut);
      umma::fence_after_sync();
      if (mine) {
        const float ai = ex2(before + pin);
        __nv_bfloat16* yp = static_cast<__nv_bfloat16*>(p.y) + ((tc0 + row) * p.H) * p.P + col;
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
          if (row < len) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              float xv[8], zv[8];
              tc::unpack8<__nv_bfloat16>(*tile16(sm + M::kX, row, half * 4 + q2 * 2 + q), xv);
              if (p.z) tc::unpack8<__nv_bfloat16>(zr[q2 * 2 + q], zv);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                float o = fmaf(D, xv[e], fmaf(ai, yi[q * 8 + e], ya[q * 8 + e]));
                if (p.z) o *= silu(zv[e]);
                xv[e] = o;
              }
              *reinterpret_cast<uint4*>(yp + q2 * 16 + q * 8) = tc::pack8<__nv_bfloat16>(xv);
            }
          }
        }
      }
      if (want_state) {  // the lowest part of w x, into the high part's tile
        wait(bar_dh, par_dh, kSiteScanState);
        par_dh ^= 1;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[8], rest[8], low[8];
          tc::unpack8<__nv_bfloat16>(*tile16(sm + M::kX, row, half * 4 + q), v);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = row < len ? v[e] * wj : 0.f;
          pack_rest(v, rest);
          pack_rest(rest, low);
          *tile16(sm + M::kXs, row, half * 4 + q) = tc::pack8<__nv_bfloat16>(low);
        }
        umma::fence_proxy_async();
        umma::fence_before_sync();
        if (__syncthreads_or(!mine)) { ok = false; break; }
        umma::fence_after_sync();
        if (tid == 0) {
          mma_dh(M::kXs, false);
          umma::mma_commit(bar_dh);
          ++commits_dh;
        }
        __syncwarp();
      }
    }
    // ---- state ----
    wait(bar_dh, par_dh, kSiteScanState);
    par_dh ^= 1;
    umma::fence_after_sync();
    // every thread is past its reads of the tiles and the products are done
    umma::fence_proxy_async();
    umma::fence_before_sync();
    if (__syncthreads_or(!mine)) { ok = false; break; }
    if (tid == 0 && c + 1 < nch) {
      fetch(c + 1);
      ++loads;
    }
    __syncwarp();
    const float decay = ex2(all);
    {
      float d[32];
      umma::tmem_ld32(tl + M::kDH + half * 32, d);
#pragma unroll
      for (int j = 0; j < 32; ++j) hr[j] = fmaf(decay, hr[j], d[j]);
    }
    if (OUT && c + 1 < nch) store_h();
    has_h = true;
    umma::fence_before_sync();
  }
  if (ok && row < S_) {
    if (OUT) {
      if (last && p.final_state)
#pragma unroll
        for (int j = 0; j < 32; ++j) st_any(p.final_state, p.final_dtype, at_seq + static_cast<int64_t>(j) * S_, hr[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) p.seg_state[at_seg + static_cast<int64_t>(j) * S_] = hr[j];
      if (tid == 0 && p0 == 0) p.seg_decay[id * p.H + h] = logd * 0.6931471805599453f;
    }
  }
  if (!ok && tid == 0) {
    // copies and products that this CTA issued may be in flight: wait
    // (bounded) for the last of each before memory is released
    const long long drain = 20000000LL;
    if (loads) umma::mbar_wait(bar_ld, (loads - 1) & 1, drain);
    if (commits_s) umma::mbar_wait(bar_s, (commits_s - 1) & 1, drain);
    if (commits_y) umma::mbar_wait(bar_y, (commits_y - 1) & 1, drain);
    if (commits_dh) umma::mbar_wait(bar_dh, (commits_dh - 1) & 1, drain);
  }
  umma::fence_before_sync();
  __syncthreads();
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

template <int S_, bool OUT>
static cudaError_t launch_kernel(const ScanParams& p, int slices, const CUtensorMap& tx, const CUtensorMap& tb,
                                 const CUtensorMap& tcm, cudaStream_t s) {
  auto kern = scan_tc_kernel<S_, OUT>;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<S_, OUT>::kBytes);
  if (e != cudaSuccess) return e;
  note_launch();
  kern<<<static_cast<unsigned>(p.segments * p.H * slices), kTcThreads, Smem<S_, OUT>::kBytes, s>>>(p, slices, tx, tb, tcm);
  return cudaGetLastError();
}

template <int S_>
static cudaError_t run_tc(ScanParams p, const gdn_scan_args& a, cudaStream_t s) {
  CUtensorMap tx, tb, tcm;
  cudaError_t e;
  const int64_t total = a.B * a.T, gs = static_cast<int64_t>(a.G) * a.S;
  if ((e = make_rows_map(&tx, a.x, static_cast<int64_t>(a.H) * a.P, total, a.stride_x)) != cudaSuccess) return e;
  if ((e = make_rows_map(&tb, a.b, gs, total, a.stride_b)) != cudaSuccess) return e;
  if ((e = make_rows_map(&tcm, a.c, gs, total, a.stride_c)) != cudaSuccess) return e;
  const int slices = a.P / 64;
  if (p.seg_state) {
    if ((e = launch_kernel<S_, false>(p, slices, tx, tb, tcm, s)) != cudaSuccess) return e;
    launch_pass(p, s);
    p.clear_err = 0;
  }
  return launch_kernel<S_, true>(p, slices, tx, tb, tcm, s);
}

cudaError_t launch_tc(const ScanParams& p, const gdn_scan_args& a, cudaStream_t s) {
  if (p.segments * p.H * (a.P / 64) > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  return a.S == 128 ? run_tc<128>(p, a, s) : run_tc<64>(p, a, s);
}

}  // namespace scan
}  // namespace gdn
