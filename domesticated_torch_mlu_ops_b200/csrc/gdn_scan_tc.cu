// Selective scan over prompts on the tensor cores (tcgen05), bf16.
//
// A small kernel first turns the raw steps into what the tiles need per token
// and head: a_i, the log2 decay from the start of the token's block of 32 to
// it, k_i = dt'_i times the decay from it to the block's end, and the log2
// decays over whole blocks (scan_prep_kernel).
//
// scan_tc_kernel: one CTA per (segment of a sequence, head, 64 columns of P),
// one per SM: sixteen warps that share the elementwise work and one that
// issues copies and products.  It walks the segment in chunks of 128 tokens:
//   S  = C B^T                                   [128, 128]
//   Yi = C h                                     [128, 64]
//   P_ij = S_ij decay(j to i) dt'_j  (j <= i),   P_ii += D
//   Ya = P x;   y = decay(to i) Yi + Ya          in fp32, then the gate
//   dH = B^T (w x),  w_j = decay(j to the end) dt'_j
//   h <- decay(chunk) h + dH                     fp32, in registers
// Four products with fp32 accumulators in TMEM.  P replaces the scores there
// and is Ya's operand from there; the parts of h and of w x lie side by side,
// so that Yi reads C and dH reads B once.  x, B and C come by TMA into
// 128-byte-swizzled tiles that serve as operands in both directions, each as
// soon as its place is free: B and C's first half behind the products of the
// chunk before the last, x after that chunk's y, which takes x's place and
// leaves by a TMA store.  z has room only in C's second half between Yi and
// the outputs, so it is brought to L2 a chunk ahead.  A chunk's chain is P and
// w x from the scores (which run behind the previous chunk's products), Ya and
// dH, and the new h.
//
// scan_tc_state_kernel, the first pass over split sequences: dH of a whole
// segment in one accumulator, chunks from the last to the first, each
// weighted by the decay to the segment's end.
//
// What bounds it.  The products of a chunk take about 2.5 K cycles of the
// tensor pipe (per step of 16 measured 64 at 128 columns, 93 at 192, and 32 at
// 64 with the operand in TMEM), a chunk step about 6 K: P and w x, Ya and dH
// beside the first part of the outputs, the rest of them and h, each by all
// sixteen warps.  Their work and that chain take the same time (41 % of the
// issue slots, 39 % of the tensor pipe), and shared memory leaves room for one
// CTA per SM.  64 heads of 64 x 128: 8192 tokens 21 us (first pass) and 112 us,
// with steps and hand-over 145 us for 208 MB; 31,992 packed tokens that start
// from states 422 us and 14 us of steps.  What each choice gave on those two
// when it was made: P through TMEM and one product for dH 106 -> 105 and 417 ->
// 410 us, z before the next chunk's operands and in L2 88 and 351, operands as
// their places become free 82 to 85 and 330, decays by sums 87 -> 90 and 336 ->
// 344, two parts of P and h 112 and 421.  Measured and set aside: w x and dH
// before P, so that h is ready before the outputs (1.15 times), both halves of
// the scores behind one wait, w x shared out by who has no block of P, products
// issued by a working warp (1.7 times); of the two parts' ways: P announced
// before w x (126 and 473), both parts of h into one accumulator, which reads C
// twice, y stored by the warps themselves (151 and 571: the fences wait for
// it).
//
// Rounding.  x, B and C are bf16 already.  P, h and w x are split into bf16
// parts whose products are summed: two parts (16 bits) where they only feed y,
// which is rounded to 8 bits in the end (one output in 1100 on the two prompts
// above rounds otherwise than the exact one); three (24 bits) of w x where the
// state is returned or handed on, so that a returned fp32 state has fp32
// precision.
// One part of P and h each would take 22 and 77 us less on the two prompts
// above and round a fifth of the outputs otherwise.
//
// Decays are products of sums that only add: the decay between two blocks' is
// exp(a_i + the blocks between) k_j, w is k times the blocks after.  No
// difference of long prefix sums occurs, whose rounding would stay behind a
// fast decay as the error of the slow ones after it.  Within the diagonal
// block P takes exp(a_i) kd_j with kd_j = dt'_j / exp(a_j) while no a reaches
// 100 there (kd stays in range, and the rounding of a under 2^-17); rows past
// that take the sum between the two tokens itself.  Either way it depends on
// no later token.  One exponential per row and block instead of one per
// element.

#include <cuda.h>

#include "gdn_chunk_tc.cuh"
#include "gdn_scan.h"
#include "scan_common.cuh"

namespace gdn {
namespace scan {

constexpr int kL = 128;             // tokens per chunk
constexpr int kTile = kL * 128;     // 128 rows x 128 bytes (64 bf16 columns)
constexpr int kWork = 512;          // threads of the sixteen working warps
constexpr int kTcThreads = kWork + 32;  // and the issuing warp
constexpr int kLead = kWork / 32;
constexpr long long kWaitLimit = 2000000000LL;

struct PrepOut {
  float *a, *k, *dt;  // [H][chunks][128]; past a sequence's end the step dt is 0
  float* sums;        // [H][chunks][kSums], of a over whole blocks of 32:
  int64_t chunks;
};
// before block b, after it, between block J and block I > J, and of the chunk
constexpr int kSums = 28, kBefore = 0, kAfter = 4, kBetween = 8, kWhole = 24;
constexpr int kStepBytes = 2 * kL * 4 + kSums * 4;  // a stage of a, k and the sums
constexpr float kFar = 100.f;                       // see the diagonal block above

template <int S_>
struct Smem {
  // two stages of operands
  static constexpr int kC = 0;                              // C
  static constexpr int kZ = kC + kTile;                     // z: in C's second tile, or its own (S = 64)
  static constexpr int kB = kC + 2 * kTile;
  static constexpr int kX = kB + S_ / 64 * kTile;           // x, then y
  static constexpr int kStage = kX + kTile;
  static constexpr int kXs = 2 * kStage;                    // the parts of w x
  static constexpr int kHlo = kXs + 2 * kTile;              // h's second part, in turns with the third of w x
  static constexpr int kH = kXs + 3 * kTile;                // h's first part
  static constexpr int kSc = kH + kTile;               // two stages of a, k and the sums
  static constexpr int kBar = kSc + 2 * kStepBytes;    // loads[2], S, Yi, Ya, dH, z, h ready, P and w x ready
  static constexpr int kBars = 9;
  static constexpr int kTmem = kBar + kBars * 8;
  static constexpr int kBad = kTmem + 8;                    // [2][64 columns + 1]: see the kernel
  static constexpr int kBytes = kBad + 2 * 65 * 4;
  static constexpr uint32_t kTx = (S_ / 64 * 2 + 1) * kTile + kStepBytes;
  // TMEM columns: S first (P in its place), Yi one accumulator per part of h
  // (the second part's first), dH one per part of w x
  static constexpr int kCols = 512, kYi = 128, kDH = 256, kYa = 448;
  static_assert(kBytes <= 227 * 1024, "shared memory");
};

// First pass: three stages of B (read until its products are done), two of x
// (read until it is split) and two of its three parts.
template <int S_>
struct StateSmem {
  static constexpr int kBStage = S_ / 64 * kTile;
  static constexpr int kX = 3 * kBStage;
  static constexpr int kXs = kX + 2 * kTile;
  static constexpr int kStep = (kL + kSums) * 4;
  static constexpr int kSc = kXs + 6 * kTile;   // two stages of k and the sums, with x
  static constexpr int kBar = kSc + 2 * kStep;  // B[3], x[2], parts ready[2], products[2]
  static constexpr int kTmem = kBar + 9 * 8;
  static constexpr int kBytes = kTmem + 8;
  static constexpr int kCols = 256;  // an accumulator per part
  static_assert(kBytes <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

// Steps of one chunk of 128 tokens for 16 heads per block (a 32-byte sector
// of 16-bit steps): raw steps in through shared memory (rows of heads are what
// is contiguous), a, k and dt out per head with tokens contiguous.  A warp
// scans a head's 128 tokens, four per lane, a block of 32 per eight lanes.
constexpr int kPrepHeads = 16;
__global__ void __launch_bounds__(kPrepHeads * 32) scan_prep_kernel(const ScanParams p, const PrepOut o) {
  __shared__ float raw[kL][kPrepHeads + 1];
  clear_error(p);
  zero_outside(p, 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h0 = blockIdx.y * kPrepHeads;
  int64_t n, ls, t0, t1;
  bool last;
  int64_t chunk0;
  if (!find_segment(p, blockIdx.x, n, ls, t0, t1, last, chunk0)) return;  // p.seg is the chunk here
  const int len = static_cast<int>(t1 - t0);
  {
    constexpr int kTurns = kL / (2 * kPrepHeads);  // two tokens per warp and turn, all turns' loads together
    const int hh = lane % kPrepHeads, i0 = warp * 2 + lane / kPrepHeads;
    float v[kTurns];
#pragma unroll
    for (int j = 0; j < kTurns; ++j) {
      const int i = i0 + j * 2 * kPrepHeads;
      v[j] = i < len && h0 + hh < p.H ? ld_any(p.dt, p.dt_dtype, (t0 + i) * p.sdt + h0 + hh) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kTurns; ++j) raw[i0 + j * 2 * kPrepHeads][hh] = v[j];
  }
  __syncthreads();
  if (h0 + warp < p.H) {
    const int hh = warp, h = h0 + hh;
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
    float up = pre[3], dn = suf[0] + a[0];  // lane totals -> sums over the block's earlier lanes, and its later ones
#pragma unroll
    for (int s = 1; s < 8; s <<= 1) {
      const float u = __shfl_up_sync(0xffffffffu, up, s, 8), v = __shfl_down_sync(0xffffffffu, dn, s, 8);
      if ((lane & 7) >= s) up += u;
      if ((lane & 7) + s < 8) dn += v;
    }
    up = __shfl_up_sync(0xffffffffu, up, 1, 8);
    dn = __shfl_down_sync(0xffffffffu, dn, 1, 8);
    if ((lane & 7) == 0) up = 0.f;
    if ((lane & 7) == 7) dn = 0.f;
    const int64_t chunk = h * o.chunks + blockIdx.x, at = chunk * kL + lane * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) pre[e] += up;
    *reinterpret_cast<float4*>(o.a + at) = make_float4(pre[0], pre[1], pre[2], pre[3]);
    *reinterpret_cast<float4*>(o.k + at) =
        make_float4(ex2(suf[0] + dn) * d[0], ex2(suf[1] + dn) * d[1], ex2(suf[2] + dn) * d[2], ex2(suf[3] + dn) * d[3]);
    *reinterpret_cast<float4*>(o.dt + at) = make_float4(d[0], d[1], d[2], d[3]);
    float tot[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) tot[b] = __shfl_sync(0xffffffffu, pre[3], b * 8 + 7);
    if (lane < kSums) {
      const int from = lane < kAfter ? 0 : lane < kBetween ? lane - kAfter + 1 : lane < kWhole ? (lane & 3) + 1 : 0;
      const int to = lane < kAfter ? lane : lane < kBetween ? 4 : lane < kWhole ? (lane - kBetween) >> 2 : 4;
      float v = 0.f;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (b >= from && b < to) v += tot[b];
      o.sums[chunk * kSums + lane] = v;
    }
  }
}

__device__ __forceinline__ float lds4(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}

// Byte offsets of a thread's two 16-byte pieces (columns 16 cq .. 16 cq + 15
// of 64) in row `row` of a swizzled tile.
struct Pieces {
  uint32_t at[2];
  __device__ __forceinline__ Pieces(int row, int cq) {
    at[0] = row * 128 + (((cq * 2) ^ (row & 7)) << 4);
    at[1] = at[0] ^ 16;
  }
};
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ void sts4(uint32_t a, float v) { asm volatile("st.shared.f32 [%0], %1;" :: "r"(a), "f"(v) : "memory"); }
__device__ __forceinline__ float4 lds16f(uint32_t a) {
  const uint4 v = lds16(a);
  return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
}
__device__ __forceinline__ void sts16(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" :: "r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// All of this warp's writes to shared memory, for the products: then one
// arrival per warp.
__device__ __forceinline__ void publish(uint32_t bar) {
  umma::fence_proxy_async();
  umma::fence_before_sync();
  __syncwarp();
  if (umma::elect_one()) umma::mbar_arrive(bar);
  __syncwarp();
}

// Columns of k-step ks of P's two parts in TMEM: side by side where the 16
// scores were that they came from.
__host__ __device__ constexpr uint32_t p_step(int ks, int part) { return ks * 16 + part * 8; }
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

// Where value 4 r of the diagonal block's kd is: a warp keeps them in the first
// pieces that it will write of the block's first eight rows of w x.
__device__ __forceinline__ uint32_t kd_at(uint32_t tile, int quad, int r) {
  return tile + (quad * 32 + r) * 128 + (((quad * 2) ^ r) << 4);
}

// A diagonal block of P with rows whose a, or an earlier one, is not under
// kFar: those take the sum of the steps between the two tokens.  `step` is the
// row's own log2 decay, dt its step.  Out of line: its registers would push the
// common path's out.
__device__ __noinline__ void diag_by_sums(uint32_t ts, int row, float ai, float step, float dt, float D,
                                          uint32_t tile) {
  const int lane = row & 31;
  float most = fabsf(ai) < kFar ? 0.f : 1.f;  // a NaN counts
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const float v = __shfl_up_sync(0xffffffffu, most, s);
    if (lane >= s) most = fmaxf(most, v);
  }
  const float f = ex2(ai);
  float sum = 0.f;  // of the steps after token j up to the row's
#pragma unroll 1
  for (int hf = 1; hf >= 0; --hf) {
    float v[16];
    umma::tmem_ld16(ts + hf * 16, v);
    uint4 hi[2], lo[2];
#pragma unroll
    for (int q = 3; q >= 0; --q) {
      const float4 k4 = lds16f(kd_at(tile, row >> 5, hf * 4 + q));
      const float kk[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
      for (int e = 3; e >= 0; --e) {
        const int i = q * 4 + e, j = hf * 16 + i;
        const float next = __shfl_sync(0xffffffffu, step, (j + 1) & 31), dj = __shfl_sync(0xffffffffu, dt, j);
        if (j < lane) sum += next;
        v[i] = j <= lane ? v[i] * (most == 0.f ? f * kk[e] : ex2(sum) * dj) : 0.f;
        if (j == lane) v[i] += D;
      }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      float2 w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = make_float2(v[q * 8 + e * 2], v[q * 8 + e * 2 + 1]);
      hi[q] = take_part(w);
      lo[q] = pack8(w);
    }
    umma::tmem_st8(ts + p_step(hf, 0), hi[0], hi[1]);
    umma::tmem_st8(ts + p_step(hf, 1), lo[0], lo[1]);
  }
}

// z / (1 + exp(-z)) of two values, to a few fp32 ulp.
__device__ __forceinline__ float2 silu2(float2 z) {
  const float2 t = __fmul2_rn(z, make_float2(-tc::kLog2e, -tc::kLog2e));
  const float2 u = __fadd2_rn(make_float2(ex2(t.x), ex2(t.y)), make_float2(1.f, 1.f));
  return __fmul2_rn(z, make_float2(rcp(u.x), rcp(u.y)));
}

// Non-zero when one of two bf16 values is infinite or NaN.
__device__ __forceinline__ uint32_t all_ones_exponent(uint32_t w) {
  return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}
// A thread's 16 columns of x with infinities or NaN: notes them and zeroes
// them in the operand's tile.
__device__ __forceinline__ void mark_not_finite(uint32_t tile, uint32_t at0, int* bad, int row, int chunk) {
#pragma unroll 1
  for (int e = 0; e < 16; ++e) {
    const uint32_t at = tile + (at0 ^ ((e >> 3) * 16)) + (e & 7) * 2;
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
    if ((v & 0x7f80) != 0x7f80) continue;
    asm volatile("st.shared.u16 [%0], %1;" :: "r"(at), "h"(static_cast<uint16_t>(0)) : "memory");
    atomicMax(bad + e, (chunk + 1) * 256 + 255 - row);
  }
}
// Token `row`'s outputs (in the tile, or at y) that follow a bad x: NaN.
__device__ __forceinline__ void nan_after(uint32_t tile, uint32_t at0, const int* bad, int row, int chunk, __nv_bfloat16* y) {
#pragma unroll 1
  for (int e = 0; e < 16; ++e) {
    const int v = *reinterpret_cast<const volatile int*>(bad + e);
    if ((v >> 8) != chunk + 1 || row < 255 - (v & 255)) continue;
    const uint16_t nan = 0x7fc0;
    if (y) *reinterpret_cast<uint16_t*>(y + e) = nan;
    else asm volatile("st.shared.u16 [%0], %1;" :: "r"(tile + (at0 ^ ((e >> 3) * 16)) + (e & 7) * 2), "h"(nan) : "memory");
  }
}

template <int S_>
__global__ void __launch_bounds__(kTcThreads, 1)
scan_tc_kernel(const ScanParams p, const PrepOut prep, const int slices, const __grid_constant__ CUtensorMap tx,
               const __grid_constant__ CUtensorMap tb, const __grid_constant__ CUtensorMap tcm,
               const __grid_constant__ CUtensorMap ty, const __grid_constant__ CUtensorMap tz) {
  using M = Smem<S_>;
  extern __shared__ __align__(1024) uint8_t sm[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + M::kBar);
  uint32_t* tslot = reinterpret_cast<uint32_t*>(sm + M::kTmem);
  const uint32_t sbase = umma::smem_u32(sm);
  const uint32_t bar_ld = umma::smem_u32(bars), bar_s = bar_ld + 16, bar_yi = bar_ld + 24, bar_y = bar_ld + 32,
                 bar_dh = bar_ld + 40, bar_z = bar_ld + 48, bar_h = bar_ld + 56, bar_px = bar_ld + 64;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (!base_ok(p, sbase)) return;
  // Block = segment * units + unit: the CTAs that read the same B and C are
  // adjacent and run together, so those come from L2.
  const int units = p.H * slices;
  const int64_t id = blockIdx.x / units;
  const int unit = static_cast<int>(blockIdx.x - id * units), h = unit / slices, p0 = (unit - h * slices) * 64;
  const int g = h / (p.H / p.G);
  int64_t n = 0, ls = 0, t0 = 0, t1 = 0;
  bool last = false;
  int64_t chunk0 = 0;
  if (!find_segment(p, id, n, ls, t0, t1, last, chunk0)) return;  // every warp finds the same
  const int64_t prow = (h * prep.chunks + chunk0) * kL;  // a, k, dt of the segment's first token
  const int nch = static_cast<int>((t1 - t0 + kL - 1) / kL);
  if (chunk0 + nch > prep.chunks) return;  // sequences that overlap: more chunks than tokens
  const bool want_state = last && p.final_state;
  // an all-zero state needs no product
  const bool seg = p.seg_state != nullptr, ini = !seg && p.init;
  auto length = [&](int c) { return static_cast<int>(min64(kL, t1 - t0 - static_cast<int64_t>(c) * kL)); };

  if (warp == kLead) {
    if (umma::elect_one()) {
#pragma unroll
      for (int i = 0; i < M::kBars; ++i) umma::mbar_init(bars + i, i < 7 ? 1 : kLead);
      umma::mbar_fence_init();
    }
    __syncwarp();
    umma::tmem_alloc(tslot, M::kCols);
    umma::fence_before_sync();
  }
  // An infinite or NaN x would reach earlier tokens of its chunk through P's
  // zeros.  It is 0 as Ya's operand, and its column's outputs from its token on
  // are NaN: bad[chunk parity][column] = (chunk + 1) * 256 + 255 - first such
  // token, and [64] the last chunk that has any.
  int* bad = reinterpret_cast<int*>(sm + M::kBad);
  if (tid < 2 * 65) bad[tid] = 0;
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tslot, 0);

  bool mine = true;
  auto wait = [&](uint32_t bar, uint32_t parity, int site) {
    // one answer per warp: what follows holds warp-wide instructions
    const bool got = __all_sync(0xffffffffu, mine && (umma::mbar_test(bar, parity) || umma::mbar_wait(bar, parity, kWaitLimit)));
    if (mine && !got) record_device_error(p.err, kErrWaitTimeout, site, static_cast<int>(blockIdx.x), tid);
    mine = got;
    return got;
  };

  if (warp == kLead) {
    // ---- copies and products ----
    constexpr uint32_t id_s = umma::idesc_f16(128, 128, true, false, false);
    constexpr uint32_t id_y = umma::idesc_f16(128, 64, true, false, true), id_yi = umma::idesc_f16(128, 128, true, false, true);
    constexpr uint32_t id_h2 = umma::idesc_f16(128, 128, true, true, true), id_h3 = umma::idesc_f16(128, 192, true, true, true);
    // operand descriptors: rows of x and of the parts are tokens (K) with 64
    // columns (N), B is read both ways; a k-step of 16 advances 32 bytes
    // within a K-major atom of 64 columns and 2048 bytes over MN-major rows
    const uint64_t d_c = umma::smem_desc_sw128(sbase + M::kC, 16, 1024), d_bk = umma::smem_desc_sw128(sbase + M::kB, 16, 1024);
    const uint64_t d_bm = umma::smem_desc_sw128(sbase + M::kB, kTile, 1024), d_x = umma::smem_desc_sw128(sbase + M::kX, kTile, 1024);
    const uint64_t d_xs = umma::smem_desc_sw128(sbase + M::kXs, kTile, 1024);
    const uint64_t d_h = umma::smem_desc_sw128(sbase + M::kHlo, kTile, 1024);  // both parts side by side
    // a chunk's operands in the order in which their places become free: B and
    // C's first tile with the products of the chunk before the last, C's
    // second tile (where z was) and x (where y was) with its outputs
    auto load_c = [&](int c, int q) {
      umma::tma_load_2d(sm + (c & 1) * M::kStage + M::kC + q * kTile, &tcm, g * S_ + q * 64, static_cast<int>(t0) + c * kL,
                        bar_ld + (c & 1) * 8);
    };
    auto fetch_bc = [&](int c) {
      const uint32_t bar = bar_ld + (c & 1) * 8;
      umma::mbar_arrive_expect_tx(bar, M::kTx);
      uint8_t* sc = sm + M::kSc + (c & 1) * kStepBytes;
      umma::bulk_g2s(sc, prep.a + prow + c * kL, kL * 4, bar);
      umma::bulk_g2s(sc + kL * 4, prep.k + prow + c * kL, kL * 4, bar);
      umma::bulk_g2s(sc + 2 * kL * 4, prep.sums + (prow / kL + c) * kSums, kSums * 4, bar);
#pragma unroll
      for (int q = 0; q < S_ / 64; ++q)
        umma::tma_load_2d(sm + (c & 1) * M::kStage + M::kB + q * kTile, &tb, g * S_ + q * 64, static_cast<int>(t0) + c * kL, bar);
      load_c(c, 0);
    };
    auto fetch_c2 = [&](int c) {
      if (S_ == 128) load_c(c, 1);
    };
    auto fetch_x = [&](int c) {
      umma::tma_load_2d(sm + (c & 1) * M::kStage + M::kX, &tx, h * p.P + p0, static_cast<int>(t0) + c * kL, bar_ld + (c & 1) * 8);
    };
    // z has room only for the time between Yi and the outputs: to L2 a chunk ahead
    auto prefetch_z = [&](int c) { umma::tma_prefetch_2d(&tz, h * p.P + p0, static_cast<int>(t0) + c * kL); };
    auto fetch_z = [&](int c) {
      umma::mbar_arrive_expect_tx(bar_z, kTile);
      umma::tma_load_2d(sm + (c & 1) * M::kStage + M::kZ, &tz, h * p.P + p0, static_cast<int>(t0) + c * kL, bar_z);
    };
    auto store_y = [&](int c) {
      umma::tma_store_2d(&ty, sm + (c & 1) * M::kStage + M::kX, h * p.P + p0, static_cast<int>(t0) + c * kL);
      umma::bulk_commit();
    };
    auto scores = [&](int c) {
      const uint64_t st = (c & 1) * (M::kStage >> 4);
#pragma unroll
      for (int ks = 0; ks < S_ / 16; ++ks)
        umma::mma_f16(tmem, d_c + st + k_step(ks), d_bk + st + k_step(ks), id_s, ks > 0);
      umma::mma_commit(bar_s);
    };
    int loads = 0, n_s = 0, n_yi = 0, n_y = 0, n_dh = 0, n_z = 0;  // issued so far
    if (nch > 0) {
      if (umma::elect_one()) {
        for (int c = 0; c < min(nch, 2); ++c) {
          fetch_bc(c);
          fetch_c2(c);
          fetch_x(c);
          if (p.z && c == 0) prefetch_z(0);
        }
      }
      __syncwarp();
      loads = min(nch, 2);
      if (wait(bar_ld, 0, kSiteScanLoad)) {
        if (umma::elect_one()) scores(0);
        __syncwarp();
        n_s = 1;
      }
    }
    for (int c = 0; c < nch && mine; ++c) {
      // h of this chunk is in place, and all work on the chunk before is done
      if (!wait(bar_h, c & 1, kSiteScanState)) break;
      umma::fence_after_sync();
      if (umma::elect_one()) {
        if (c > 0) store_y(c - 1);  // a whole chunk
        if (c > 0 && c + 1 < nch) fetch_c2(c + 1);
        const uint64_t st = (c & 1) * (M::kStage >> 4);
        if (c > 0 || seg || ini)
#pragma unroll
          for (int ks = 0; ks < S_ / 16; ++ks)
            umma::mma_f16(tmem + M::kYi, d_c + st + k_step(ks), d_h + mn_step(ks), id_yi, ks > 0);
        umma::mma_commit(bar_yi);
        if (c > 0 && c + 1 < nch) {
          umma::bulk_wait_read_all();
          fetch_x(c + 1);
        }
      }
      __syncwarp();
      ++n_yi;
      if (p.z) {  // in C's second tile once Yi has read it
        if (!wait(bar_yi, c & 1, kSiteScanScores)) break;
        if (umma::elect_one()) {
          fetch_z(c);
          if (c + 1 < nch) prefetch_z(c + 1);
        }
        __syncwarp();
        ++n_z;
      }
      if (!wait(bar_px, c & 1, kSiteScanScores)) break;
      umma::fence_after_sync();
      if (umma::elect_one()) {
        const uint64_t st = (c & 1) * (M::kStage >> 4);
#pragma unroll
        for (int ks = 0; ks < kL / 16; ++ks)
          umma::mma_f16_ta(tmem + M::kYa, tmem + p_step(ks, 0), d_x + st + mn_step(ks), id_y, ks > 0);
#pragma unroll
        for (int ks = 0; ks < kL / 16; ++ks)  // the parts in turns, step by step, took 19 us longer over 32 chunks
          umma::mma_f16_ta(tmem + M::kYa, tmem + p_step(ks, 1), d_x + st + mn_step(ks), id_y, 1);
        umma::mma_commit(bar_y);
        // The parts of w x side by side: one product reads B once for all.
        // With S = 64 rows 64-127 of the accumulators are the product of the
        // tile after B: never read.
        const uint32_t id_h = want_state ? id_h3 : id_h2;
#pragma unroll
        for (int ks = 0; ks < kL / 16; ++ks)
          umma::mma_f16(tmem + M::kDH, d_bm + st + mn_step(ks), d_xs + mn_step(ks), id_h, ks > 0);
        umma::mma_commit(bar_dh);
      }
      __syncwarp();
      ++n_y;
      ++n_dh;
      if (c + 1 < nch) {
        if (!wait(bar_ld + ((c + 1) & 1) * 8, ((c + 1) >> 1) & 1, kSiteScanLoad)) break;
        if (!wait(bar_y, c & 1, kSiteScanOut)) break;  // P is read: the scores take its place
        umma::fence_after_sync();
        if (umma::elect_one()) scores(c + 1);
        __syncwarp();
        ++n_s;
        if (c + 2 < nch) {
          if (!wait(bar_dh, c & 1, kSiteScanState)) break;
          if (umma::elect_one()) fetch_bc(c + 2);
          __syncwarp();
          ++loads;
        }
      }
    }
    if (mine && nch > 0 && wait(bar_h, nch & 1, kSiteScanState)) {  // the last chunk's y
      if (umma::elect_one() && length(nch - 1) == kL) store_y(nch - 1);
    }
    __syncwarp();
    if (umma::elect_one()) umma::bulk_wait_all();
    __syncwarp();
    if (!mine) {
      // copies and products that were issued may be in flight: wait (bounded)
      // for the last of each before memory is released
      const long long drain = 20000000LL;
      if (loads > 1) umma::mbar_wait(bar_ld + (loads & 1) * 8, ((loads - 2) >> 1) & 1, drain);
      if (loads > 0) umma::mbar_wait(bar_ld + ((loads - 1) & 1) * 8, ((loads - 1) >> 1) & 1, drain);
      if (n_z) umma::mbar_wait(bar_z, (n_z - 1) & 1, drain);
      if (n_s) umma::mbar_wait(bar_s, (n_s - 1) & 1, drain);
      if (n_yi) umma::mbar_wait(bar_yi, (n_yi - 1) & 1, drain);
      if (n_y) umma::mbar_wait(bar_y, (n_y - 1) & 1, drain);
      if (n_dh) umma::mbar_wait(bar_dh, (n_dh - 1) & 1, drain);
    }
  } else {
    // ---- everything between the products ----
    const int quad = warp & 3, cq = warp >> 2;  // TMEM lane quadrant; quarter of the columns
    const int row = quad * 32 + lane;           // token of the chunk, or state column s
    const uint32_t tl = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const Pieces piece(row, cq);
    const int64_t col = static_cast<int64_t>(h) * p.P + p0 + cq * 16;
    auto state_at = [&](int64_t i) { return ((i * p.H + h) * p.P + p0 + cq * 16) * S_ + row; };
    const float D = p.D ? p.D[h] : 0.f;
    float dt_next = 0.f;  // of the diagonal block, loaded a chunk ahead
    if (cq == quad && nch > 0) dt_next = __ldg(prep.dt + prow + row);
    float2 hr[8];  // h[s = row][16 columns of P]
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float v = 0.f;
      if (row < S_) {
        if (seg) v = p.seg_state[state_at(id * p.subs) + j * S_];
        else if (ini) v = ld_any(p.init, p.init_dtype, state_at(n) + j * S_);
      }
      if (j & 1) hr[j / 2].y = v;
      else hr[j / 2].x = v;
    }
    auto store_h = [&]() {
      if (row < S_) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float2 v[4] = {hr[q * 4], hr[q * 4 + 1], hr[q * 4 + 2], hr[q * 4 + 3]};
          sts16(sbase + M::kH + piece.at[q], take_part(v));
          sts16(sbase + M::kHlo + piece.at[q], pack8(v));
        }
      }
    };
    store_h();
    publish(bar_h);
    for (int c = 0; c < nch; ++c) {
      const int len = length(c);
      const uint32_t st = sbase + (c & 1) * M::kStage;
      const uint32_t sc_at = sbase + M::kSc + (c & 1) * kStepBytes;
      const float dt = dt_next;
      if (cq == quad && c + 1 < nch) dt_next = __ldg(prep.dt + prow + (c + 1) * kL + row);
      if (!wait(bar_ld + (c & 1) * 8, (c >> 1) & 1, kSiteScanLoad)) break;
      const uint32_t sums_at = sc_at + 2 * kL * 4;
      const float ai = lds4(sc_at + row * 4), wj = lds4(sc_at + (kL + row) * 4) * ex2(lds4(sums_at + (kAfter + quad) * 4));
      const float g1 = ex2(lds4(sums_at + (kBefore + quad) * 4) + ai), decay = ex2(lds4(sums_at + kWhole * 4));
      // ---- P from the scores: block of columns J = cq ----
      if (cq == quad) {
        sts4(kd_at(sbase + M::kXs, quad, lane >> 2) + (lane & 3) * 4, ex2(-ai) * dt);
        __syncwarp();
      }
      if (!wait(bar_s, c & 1, kSiteScanScores)) break;
      umma::fence_after_sync();
      const uint32_t ts = tl + cq * 32;
      if (cq <= quad) {
        const bool diag = cq == quad;
        if (!diag || __all_sync(0xffffffffu, fabsf(ai) < kFar)) {
          const uint32_t cf = sc_at + (kL + cq * 32) * 4;
          const float f = ex2(diag ? ai : ai + lds4(sums_at + (kBetween + quad * 4 + cq) * 4));
          const float2 f2 = make_float2(f, f);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {  // 16 columns at a time: registers
            float v[16];
            uint4 hi[2], lo[2];
            umma::tmem_ld16(ts + hf * 16, v);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int r = hf * 4 + q * 2;
              const uint4 k0 = lds16(diag ? kd_at(sbase + M::kXs, quad, r) : cf + r * 16),
                          k1 = lds16(diag ? kd_at(sbase + M::kXs, quad, r + 1) : cf + r * 16 + 16);
              const uint32_t kk[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
              float2 w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int j = hf * 16 + q * 8 + e * 2;
                const float2 k2 = make_float2(__uint_as_float(kk[e * 2]), __uint_as_float(kk[e * 2 + 1]));
                w[e] = __fmul2_rn(make_float2(v[q * 8 + e * 2], v[q * 8 + e * 2 + 1]), __fmul2_rn(f2, k2));
                if (diag) {
                  w[e].x = j < lane ? w[e].x : j == lane ? w[e].x + D : 0.f;
                  w[e].y = j + 1 < lane ? w[e].y : j + 1 == lane ? w[e].y + D : 0.f;
                }
              }
              hi[q] = take_part(w);
              lo[q] = pack8(w);
            }
            umma::tmem_st8(ts + p_step(hf, 0), hi[0], hi[1]);  // over scores that have been read
            umma::tmem_st8(ts + p_step(hf, 1), lo[0], lo[1]);
          }
        } else {
          diag_by_sums(ts, row, ai, dt * (p.A[h] * tc::kLog2e), dt, D, sbase + M::kXs);
        }
      } else {
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int q = 0; q < 4; ++q) umma::tmem_st8(ts + q * 8, zero, zero);
      }
      // ---- w x in parts (x has been there since the scores were issued) ----
      const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
      uint32_t not_finite = 0;
      if (want_state && !wait(bar_yi, c & 1, kSiteScanScores)) break;  // the third part takes the place of h's second
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint4 u = lds16(st + M::kX + piece.at[q]);
        if (row >= len) {  // another sequence's rows: zero operands, whatever they hold
          u = zero;
          sts16(st + M::kX + piece.at[q], zero);
        }
        not_finite |= all_ones_exponent(u.x) | all_ones_exponent(u.y) | all_ones_exponent(u.z) | all_ones_exponent(u.w);
        float2 v[4];
        unpack8(u, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __fmul2_rn(v[e], make_float2(wj, wj));
        sts16(sbase + M::kXs + piece.at[q], take_part(v));
        if (want_state) {
          sts16(sbase + M::kXs + kTile + piece.at[q], take_part(v));
          sts16(sbase + M::kXs + 2 * kTile + piece.at[q], pack8(v));
        } else {
          sts16(sbase + M::kXs + kTile + piece.at[q], pack8(v));
        }
      }
      if (__any_sync(0xffffffffu, not_finite != 0)) {
        if (not_finite) mark_not_finite(st + M::kX, piece.at[0], bad + (c & 1) * 65 + cq * 16, row, c);
        if (lane == 0) atomicMax(bad + (c & 1) * 65 + 64, c + 1);
        __syncwarp();
      }
      if (row >= len)
#pragma unroll
        for (int q = 0; q < S_ / 32; ++q) {
          const int at = cq * (S_ / 32) + q;  // of S_ / 8 pieces
          sts16(st + M::kB + (at >> 3) * kTile + row * 128 + (((at & 7) ^ (row & 7)) << 4), zero);
        }
      umma::tmem_st_wait();
      publish(bar_px);
      // ---- outputs: first what does not need Ya (whose product runs now) ----
      float2 part_y[8], gz[8];
      if (!wait(bar_yi, c & 1, kSiteScanScores)) break;
      umma::fence_after_sync();
      {
        const float2 g2 = make_float2(g1, g1);
        if (c > 0 || seg || ini) {
          float lo[16], hi[16];
          umma::tmem_ld16x2(tl + M::kYi + cq * 16, tl + M::kYi + 64 + cq * 16, lo, hi);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 yi = __fadd2_rn(make_float2(hi[e * 2], hi[e * 2 + 1]), make_float2(lo[e * 2], lo[e * 2 + 1]));
            part_y[e] = __fmul2_rn(g2, yi);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) part_y[e] = make_float2(0.f, 0.f);
        }
      }
      if (p.z) {
        if (!wait(bar_z, c & 1, kSiteScanLoad)) break;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          unpack8(lds16(st + M::kZ + piece.at[q]), gz + q * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) gz[q * 4 + e] = silu2(gz[q * 4 + e]);
        }
      }
      if (!wait(bar_y, c & 1, kSiteScanOut)) break;
      umma::fence_after_sync();
      {
        float ya[16];
        umma::tmem_ld16(tl + M::kYa + cq * 16, ya);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float2 o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = q * 8 + e * 2;
            o[e] = __fadd2_rn(part_y[q * 4 + e], make_float2(ya[i], ya[i + 1]));
            if (p.z) o[e] = __fmul2_rn(o[e], gz[q * 4 + e]);
          }
          const uint4 u = pack8(o);
          if (len == kL) {
            sts16(st + M::kX + piece.at[q], u);
          } else if (row < len) {
            __nv_bfloat16* yp = static_cast<__nv_bfloat16*>(p.y) + (t0 + static_cast<int64_t>(c) * kL + row) * p.H * p.P + col;
            *reinterpret_cast<uint4*>(yp + q * 8) = u;
          }
        }
      }
      // ---- state ----
      if (!wait(bar_dh, c & 1, kSiteScanState)) break;
      umma::fence_after_sync();
      {
        const float2 decay2 = make_float2(decay, decay);
        float d[16], e[16];
        umma::tmem_ld16x2(tl + M::kDH + cq * 16, tl + M::kDH + 64 + cq * 16, d, e);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          hr[j] = __ffma2_rn(decay2, hr[j], make_float2(d[j * 2], d[j * 2 + 1]));
          hr[j] = __fadd2_rn(hr[j], make_float2(e[j * 2], e[j * 2 + 1]));
        }
        if (want_state) {
          umma::tmem_ld16(tl + M::kDH + 128 + cq * 16, d);
#pragma unroll
          for (int j = 0; j < 8; ++j) hr[j] = __fadd2_rn(hr[j], make_float2(d[j * 2], d[j * 2 + 1]));
        }
      }
      store_h();
      if (*reinterpret_cast<volatile int*>(bad + (c & 1) * 65 + 64) == c + 1 && row < len)
        nan_after(st + M::kX, piece.at[0], bad + (c & 1) * 65 + cq * 16, row, c,
                  len == kL ? nullptr : static_cast<__nv_bfloat16*>(p.y) + (t0 + static_cast<int64_t>(c) * kL + row) * p.H * p.P + col);
      publish(bar_h);
    }
    if (mine && row < S_ && want_state)
#pragma unroll
      for (int j = 0; j < 16; ++j)
        st_any(p.final_state, p.final_dtype, state_at(n) + j * S_, j & 1 ? hr[j / 2].y : hr[j / 2].x);
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  if (warp == kLead) umma::tmem_dealloc(tmem, M::kCols);
}

// Block = (segment * subs + piece of it) * units + unit.
template <int S_>
__global__ void __launch_bounds__(kTcThreads, 1)
scan_tc_state_kernel(const ScanParams p, const PrepOut prep, const int slices, const __grid_constant__ CUtensorMap tx,
                     const __grid_constant__ CUtensorMap tb) {
  using M = StateSmem<S_>;
  extern __shared__ __align__(1024) uint8_t sm[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + M::kBar);
  uint32_t* tslot = reinterpret_cast<uint32_t*>(sm + M::kTmem);
  const uint32_t sbase = umma::smem_u32(sm);
  const uint32_t bar_b = umma::smem_u32(bars), bar_x = bar_b + 24, bar_xs = bar_b + 40, bar_dh = bar_b + 56;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (!base_ok(p, sbase)) return;
  const int units = p.H * slices;
  const int64_t piece_id = blockIdx.x / units, id = piece_id / p.subs;
  const int unit = static_cast<int>(blockIdx.x - piece_id * units), h = unit / slices, p0 = (unit - h * slices) * 64;
  const int g = h / (p.H / p.G);
  int64_t n = 0, ls = 0, t0 = 0, t1 = 0;
  bool last = false;
  int64_t chunk0 = 0;
  if (!find_segment(p, id, n, ls, t0, t1, last, chunk0) || last) return;
  const int64_t prow = (h * prep.chunks + chunk0) * kL + (piece_id - id * p.subs) * p.sub;
  t0 += (piece_id - id * p.subs) * p.sub;  // a segment that is not the last is whole: pieces of whole chunks
  t1 = min64(t1, t0 + p.sub);
  const int nch = static_cast<int>((t1 - t0) / kL);
  if (prow / kL + nch > (h + 1) * prep.chunks) return;  // sequences that overlap: more chunks than tokens
  if (warp == kLead) {
    if (umma::elect_one()) {
#pragma unroll
      for (int i = 0; i < 9; ++i) umma::mbar_init(bars + i, i == 5 || i == 6 ? kLead : 1);
      umma::mbar_fence_init();
    }
    __syncwarp();
    umma::tmem_alloc(tslot, M::kCols);
    umma::fence_before_sync();
  }
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tslot, 0);
  bool mine = true;
  auto wait = [&](uint32_t bar, uint32_t parity, int site) {
    const bool got = __all_sync(0xffffffffu, mine && (umma::mbar_test(bar, parity) || umma::mbar_wait(bar, parity, kWaitLimit)));
    if (mine && !got) record_device_error(p.err, kErrWaitTimeout, site, static_cast<int>(blockIdx.x), tid);
    mine = got;
    return got;
  };
  // step i works on chunk nch - 1 - i
  if (warp == kLead) {
    constexpr uint32_t id_h = umma::idesc_f16(128, 192, true, true, true);
    const uint64_t d_b = umma::smem_desc_sw128(sbase, kTile, 1024), d_xs = umma::smem_desc_sw128(sbase + M::kXs, kTile, 1024);
    auto token = [&](int i) { return static_cast<int>(t0) + (nch - 1 - i) * kL; };
    auto fetch_b = [&](int i) {
      umma::mbar_arrive_expect_tx(bar_b + (i % 3) * 8, M::kBStage);
#pragma unroll
      for (int q = 0; q < S_ / 64; ++q)
        umma::tma_load_2d(sm + (i % 3) * M::kBStage + q * kTile, &tb, g * S_ + q * 64, token(i), bar_b + (i % 3) * 8);
    };
    auto fetch_x = [&](int i) {
      const uint32_t bar = bar_x + (i & 1) * 8;
      uint8_t* sc = sm + M::kSc + (i & 1) * M::kStep;
      umma::mbar_arrive_expect_tx(bar, kTile + M::kStep);
      umma::bulk_g2s(sc, prep.k + prow + (nch - 1 - i) * kL, kL * 4, bar);
      umma::bulk_g2s(sc + kL * 4, prep.sums + (prow / kL + nch - 1 - i) * kSums, kSums * 4, bar);
      umma::tma_load_2d(sm + M::kX + (i & 1) * kTile, &tx, h * p.P + p0, token(i), bar);
    };
    if (umma::elect_one()) {
      fetch_x(0);
      fetch_b(0);
      if (nch > 1) {
        fetch_x(1);
        fetch_b(1);
      }
    }
    __syncwarp();
    int loads_b = min(nch, 2), loads_x = min(nch, 2), done = 0;
    for (int i = 0; i < nch; ++i) {
      if (!wait(bar_xs + (i & 1) * 8, (i >> 1) & 1, kSiteScanScores)) break;
      if (i + 2 < nch) {
        if (umma::elect_one()) fetch_x(i + 2);  // x of step i is split
        __syncwarp();
        ++loads_x;
        if (i > 0 && !wait(bar_dh + ((i - 1) & 1) * 8, ((i - 1) >> 1) & 1, kSiteScanState)) break;
        if (umma::elect_one()) fetch_b(i + 2);  // where step i - 1's was
        __syncwarp();
        ++loads_b;
      }
      if (!wait(bar_b + (i % 3) * 8, (i / 3) & 1, kSiteScanLoad)) break;
      umma::fence_after_sync();
      if (umma::elect_one()) {
        const uint64_t db = d_b + (i % 3) * (M::kBStage >> 4), dx = d_xs + (i & 1) * ((3 * kTile) >> 4);
#pragma unroll
        for (int ks = 0; ks < kL / 16; ++ks) umma::mma_f16(tmem, db + mn_step(ks), dx + mn_step(ks), id_h, i > 0 || ks > 0);
        umma::mma_commit(bar_dh + (i & 1) * 8);
      }
      __syncwarp();
      ++done;
    }
    if (!mine) {
      const long long drain = 20000000LL;
      for (int i = max(0, loads_b - 3); i < loads_b; ++i) umma::mbar_wait(bar_b + (i % 3) * 8, (i / 3) & 1, drain);
      for (int i = max(0, loads_x - 2); i < loads_x; ++i) umma::mbar_wait(bar_x + (i & 1) * 8, (i >> 1) & 1, drain);
      for (int i = max(0, done - 2); i < done; ++i) umma::mbar_wait(bar_dh + (i & 1) * 8, (i >> 1) & 1, drain);
    }
  } else {
    const int quad = warp & 3, cq = warp >> 2, row = quad * 32 + lane;
    const Pieces piece(row, cq);
    float later = 0.f;  // log2 decay from the chunk's end to the piece's
    for (int i = 0; i < nch; ++i) {
      const uint32_t xt = sbase + M::kX + (i & 1) * kTile, xs = sbase + M::kXs + (i & 1) * 3 * kTile;
      if (!wait(bar_x + (i & 1) * 8, (i >> 1) & 1, kSiteScanLoad)) break;
      const uint32_t sc_at = sbase + M::kSc + (i & 1) * M::kStep;
      const uint32_t sums_at = sc_at + kL * 4;
      const float wj = lds4(sc_at + row * 4) * ex2(lds4(sums_at + (kAfter + quad) * 4)) * ex2(later);
      later += lds4(sums_at + kWhole * 4);
      if (i >= 2 && !wait(bar_dh + (i & 1) * 8, ((i - 2) >> 1) & 1, kSiteScanState)) break;  // the parts' tiles are read
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float2 v[4];
        unpack8(lds16(xt + piece.at[q]), v);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __fmul2_rn(v[e], make_float2(wj, wj));
        sts16(xs + piece.at[q], take_part(v));
        sts16(xs + kTile + piece.at[q], take_part(v));
        sts16(xs + 2 * kTile + piece.at[q], pack8(v));
      }
      publish(bar_xs + (i & 1) * 8);
    }
    // the last step's products come after all others; the phase before its own
    // on that barrier was waited for above
    const int i = nch - 1;
    if (mine && wait(bar_dh + (i & 1) * 8, (i >> 1) & 1, kSiteScanState)) {
      umma::fence_after_sync();
      const uint32_t at = tmem + (static_cast<uint32_t>(quad * 32) << 16) + cq * 16;
      float d[16], e[16], f[16];
      umma::tmem_ld16x2(at, at + 64, d, e);
      umma::tmem_ld16(at + 128, f);
      if (row < S_) {
        float* out = p.seg_state + ((piece_id * p.H + h) * p.P + p0 + cq * 16) * S_ + row;
#pragma unroll
        for (int j = 0; j < 16; ++j) out[j * S_] = d[j] + (e[j] + f[j]);
      }
      if (tid == 0 && p0 == 0) p.seg_decay[piece_id * p.H + h] = later * 0.6931471805599453f;
    }
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  if (warp == kLead) umma::tmem_dealloc(tmem, M::kCols);
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

// Chunks of 128 tokens: every sequence has at most ceil(len / 128), and at least one.
static int64_t prep_chunks(const gdn_scan_args& a) { return a.B * a.T / kL + a.N; }
size_t tc_scratch_bytes(const gdn_scan_args& a) {
  return static_cast<size_t>(prep_chunks(a)) * a.H * (3 * kL + kSums) * sizeof(float);
}

template <int S_>
static cudaError_t run_tc(ScanParams p, const gdn_scan_args& a, float* scratch, cudaStream_t s) {
  CUtensorMap tx, tb, tcm, ty, tz;
  cudaError_t e;
  const int64_t total = a.B * a.T, gs = static_cast<int64_t>(a.G) * a.S, hp = static_cast<int64_t>(a.H) * a.P;
  if ((e = make_rows_map(&tx, a.x, hp, total, a.stride_x)) != cudaSuccess) return e;
  if ((e = make_rows_map(&tb, a.b, gs, total, a.stride_b)) != cudaSuccess) return e;
  if ((e = make_rows_map(&tcm, a.c, gs, total, a.stride_c)) != cudaSuccess) return e;
  if ((e = make_rows_map(&ty, a.y, hp, total, hp)) != cudaSuccess) return e;
  if ((e = make_rows_map(&tz, a.z ? a.z : a.y, hp, total, a.z ? a.stride_z : hp)) != cudaSuccess) return e;
  const int slices = a.P / 64;
  const int64_t chunks = prep_chunks(a), each = chunks * kL * a.H;
  const PrepOut prep{scratch, scratch + each, scratch + 2 * each, scratch + 3 * each, chunks};
  ScanParams q = p;
  q.seg = kL;
  note_launch();
  scan_prep_kernel<<<dim3(static_cast<unsigned>(chunks), static_cast<unsigned>((a.H + kPrepHeads - 1) / kPrepHeads)),
                     kPrepHeads * 32, 0, s>>>(
      q, prep);
  const unsigned grid = static_cast<unsigned>(p.segments * p.H * slices);
  if (p.seg_state) {
    auto kern = scan_tc_state_kernel<S_>;
    if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, StateSmem<S_>::kBytes)) != cudaSuccess)
      return e;
    note_launch();
    kern<<<grid * p.subs, kTcThreads, StateSmem<S_>::kBytes, s>>>(p, prep, slices, tx, tb);
    launch_pass(p, s);
  }
  auto kern = scan_tc_kernel<S_>;
  if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<S_>::kBytes)) != cudaSuccess)
    return e;
  note_launch();
  kern<<<grid, kTcThreads, Smem<S_>::kBytes, s>>>(p, prep, slices, tx, tb, tcm, ty, tz);
  return cudaGetLastError();
}

cudaError_t launch_tc(const ScanParams& p, const gdn_scan_args& a, float* scratch, cudaStream_t s) {
  if (p.segments * p.subs * p.H * (a.P / 64) > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  return a.S == 128 ? run_tc<128>(p, a, scratch, s) : run_tc<64>(p, a, scratch, s);
}

}  // namespace scan
}  // namespace gdn
