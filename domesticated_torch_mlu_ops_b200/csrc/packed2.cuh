// Small fp32 vectors kept as register pairs, so that every operation on an
// even length is one packed instruction per two lanes and no moves are needed
// to build the pairs; length 1 is a plain float.
#pragma once

#include "conv_math.cuh"
#include "gdn_common.cuh"

namespace gdn {
namespace pk {

template <int VEC>
struct Vec {
  static_assert(VEC % 2 == 0, "pairs");
  float2 p[VEC / 2];
};
template <>
struct Vec<1> {
  float s;
};

#define GDN_PK_LOOP _Pragma("unroll") for (int i = 0; i < VEC / 2; ++i)

template <int VEC>
__device__ __forceinline__ Vec<VEC> splat(float x) {
  Vec<VEC> r;
  if constexpr (VEC == 1) r.s = x;
  else GDN_PK_LOOP r.p[i] = make_float2(x, x);
  return r;
}
template <int VEC>
__device__ __forceinline__ Vec<VEC> fma(const Vec<VEC>& a, const Vec<VEC>& b, const Vec<VEC>& c) {
  Vec<VEC> r;
  if constexpr (VEC == 1) r.s = fmaf(a.s, b.s, c.s);
  else GDN_PK_LOOP r.p[i] = __ffma2_rn(a.p[i], b.p[i], c.p[i]);
  return r;
}
template <int VEC>
__device__ __forceinline__ Vec<VEC> mul(const Vec<VEC>& a, const Vec<VEC>& b) {
  Vec<VEC> r;
  if constexpr (VEC == 1) r.s = a.s * b.s;
  else GDN_PK_LOOP r.p[i] = __fmul2_rn(a.p[i], b.p[i]);
  return r;
}
template <int VEC>
__device__ __forceinline__ Vec<VEC> add(const Vec<VEC>& a, const Vec<VEC>& b) {
  Vec<VEC> r;
  if constexpr (VEC == 1) r.s = a.s + b.s;
  else GDN_PK_LOOP r.p[i] = __fadd2_rn(a.p[i], b.p[i]);
  return r;
}
template <int VEC>
__device__ __forceinline__ float get(const Vec<VEC>& a, int e) {
  if constexpr (VEC == 1) return a.s;
  else return e & 1 ? a.p[e / 2].y : a.p[e / 2].x;
}
template <int VEC>
__device__ __forceinline__ void set(Vec<VEC>& a, int e, float x) {
  if constexpr (VEC == 1) a.s = x;
  else if (e & 1) a.p[e / 2].y = x;
  else a.p[e / 2].x = x;
}
template <int VEC>
__device__ __forceinline__ float sum(const Vec<VEC>& a) {
  if constexpr (VEC == 1) {
    return a.s;
  } else {
    float r = a.p[0].x + a.p[0].y;
#pragma unroll
    for (int i = 1; i < VEC / 2; ++i) r += a.p[i].x + a.p[i].y;
    return r;
  }
}

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
// 1 / (1 + exp(-x)) for results of type T, two special-function instructions
// per lane; 0 and 1 at the ends.  exp(-x) = 2^t with t = -x log2(e): rounding t
// to fp32 costs 2^-24 |t| of the result, which 16 bits do not see; for fp32
// the rest of t, and of log2(e), comes back as a factor 1 + rest ln(2), so that
// a few ulp are left for every x.
template <typename T, int VEC>
__device__ __forceinline__ Vec<VEC> sigmoid(const Vec<VEC>& x) {
  constexpr float kNegLog2e = -1.4426950408889634f, kNegLog2eRest = -1.9259630e-8f, kLn2 = 0.69314718f;
  const Vec<VEC> c = splat<VEC>(kNegLog2e), t = mul(x, c);
  Vec<VEC> e, r;
#pragma unroll
  for (int i = 0; i < VEC; ++i) set(e, i, ex2(get(t, i)));
  if constexpr (sizeof(T) == 4) {
    const Vec<VEC> rest = fma(x, splat<VEC>(kNegLog2eRest), fma(x, c, mul(t, splat<VEC>(-1.f))));
    const Vec<VEC> f = fma(e, mul(rest, splat<VEC>(kLn2)), e);
#pragma unroll
    for (int i = 0; i < VEC; ++i) set(e, i, get(t, i) < 127.f ? get(f, i) : get(e, i));  // infinite, or a NaN
  }
  e = add(e, splat<VEC>(1.f));
#pragma unroll
  for (int i = 0; i < VEC; ++i) set(r, i, rcp(get(e, i)));
  return r;
}

// VEC elements of T as they lie in memory, moved by the widest instruction
// that fits; loads stay where they are written (the compiler moves plain ones
// down to their use, past the work they should overlap).
template <int BYTES>
struct Bits;
template <> struct Bits<32> { uint4 a, b; };
template <> struct Bits<16> { uint4 a; };
template <> struct Bits<8> { uint2 a; };
template <> struct Bits<4> { uint32_t a; };
template <> struct Bits<2> { uint16_t a; };

__device__ __forceinline__ void ldg_now(uint4& v, const void* p) {
  asm volatile("ld.global.nc.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
}
__device__ __forceinline__ void ldg_now(uint2& v, const void* p) {
  asm volatile("ld.global.nc.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
}
__device__ __forceinline__ void ldg_now(uint32_t& v, const void* p) {
  asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(v) : "l"(p));
}
__device__ __forceinline__ void ldg_now(uint16_t& v, const void* p) {
  asm volatile("ld.global.nc.b16 %0, [%1];" : "=h"(v) : "l"(p));
}
// The same from memory that the kernel may write later: ordinary loads, which
// stay before the stores that follow them.
__device__ __forceinline__ void ld_now(uint4& v, const void* p) {
  asm volatile("ld.global.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
}
__device__ __forceinline__ void ld_now(uint2& v, const void* p) {
  asm volatile("ld.global.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
}
__device__ __forceinline__ void ld_now(uint32_t& v, const void* p) {
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
}
__device__ __forceinline__ void ld_now(uint16_t& v, const void* p) {
  asm volatile("ld.global.b16 %0, [%1];" : "=h"(v) : "l"(p) : "memory");
}
template <typename T, int VEC>
using Raw = Bits<VEC * sizeof(T)>;
template <int BYTES>
__device__ __forceinline__ void load(Bits<BYTES>& v, const void* p) {
  ldg_now(v.a, p);
  if constexpr (BYTES == 32) ldg_now(v.b, static_cast<const char*>(p) + 16);
}
template <int BYTES>
__device__ __forceinline__ void load_rw(Bits<BYTES>& v, const void* p) {
  ld_now(v.a, p);
  if constexpr (BYTES == 32) ld_now(v.b, static_cast<const char*>(p) + 16);
}

// 32 bytes in one access, where the address is a multiple of 32.
__device__ __forceinline__ void load_rw_wide(Bits<32>& v, const void* p) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v.a.x), "=r"(v.a.y), "=r"(v.a.z), "=r"(v.a.w), "=r"(v.b.x), "=r"(v.b.y), "=r"(v.b.z), "=r"(v.b.w)
               : "l"(p) : "memory");
}
__device__ __forceinline__ void store_wide(void* p, const Bits<32>& v) {
  asm volatile("st.global.v8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};"
               :: "r"(v.a.x), "r"(v.a.y), "r"(v.a.z), "r"(v.a.w), "r"(v.b.x), "r"(v.b.y), "r"(v.b.z), "r"(v.b.w), "l"(p)
               : "memory");
}

template <typename T, int VEC>
__device__ __forceinline__ Vec<VEC> widen(const Raw<T, VEC>& v) {
  Vec<VEC> r;
  if constexpr (VEC == 1) {
    r.s = to_f<T>(reinterpret_cast<const T&>(v.a));
  } else if constexpr (sizeof(T) == 4) {
    const float2* f = reinterpret_cast<const float2*>(&v);
    GDN_PK_LOOP r.p[i] = f[i];
  } else {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(&v);
    GDN_PK_LOOP r.p[i] = conv::unpack2<T>(u[i]);
  }
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, const Vec<VEC>& a) {
  if constexpr (VEC == 1) {
    *p = from_f<T>(a.s);
  } else {
    Raw<T, VEC> v;
    if constexpr (sizeof(T) == 4) {
      float2* f = reinterpret_cast<float2*>(&v);
      GDN_PK_LOOP f[i] = a.p[i];
    } else {
      uint32_t* u = reinterpret_cast<uint32_t*>(&v);
      GDN_PK_LOOP {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(a.p[i].x, a.p[i].y);
          u[i] = *reinterpret_cast<const uint32_t*>(&b);
        } else {
          const __half2 b = __floats2half2_rn(a.p[i].x, a.p[i].y);
          u[i] = *reinterpret_cast<const uint32_t*>(&b);
        }
      }
    }
    if constexpr (VEC * sizeof(T) == 32) {
      reinterpret_cast<uint4*>(p)[0] = v.a;
      reinterpret_cast<uint4*>(p)[1] = v.b;
    } else {
      *reinterpret_cast<decltype(v.a)*>(p) = v.a;
    }
  }
}

#undef GDN_PK_LOOP

}  // namespace pk
}  // namespace gdn
