// Warp-level pieces that the attention-side kernels share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx.cuh"

namespace chord {

// The operators of a token's way through a layer are launched with the programmatic stream-serialization
// attribute, whatever the option: they are a few microseconds each, follow one another, and touch no memory before
// they have waited for what was launched before them.  us of a call among others of its kind, without and with it:
// one row of 4096 x 7168 8.3 and 6.1, 13 rows of 7168 x 2048 8.2 and 5.7, attention over 333 tokens 10.3 and
// 8.5.  They do not let the next one in before they end (attention then took 2 % longer, the others as long).
constexpr bool kEarlyLaunch = true;

// a * b + c on two BF16 numbers, rounded once.  Subnormal operands count in full, which is what
// turns bits into numbers below: a BF16 pattern under 0x100 is the number pattern * 2^-133, so a code
// of up to eight bits is a number as it stands, and one multiply-add takes its offset off.
__device__ __forceinline__ uint32_t bf16x2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

constexpr uint32_t kTwo127 = 0x7F007F00u;    // 2^127, twice

__device__ __forceinline__ float bf16_lo(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t pair) { return __uint_as_float(pair & 0xFFFF0000u); }

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Loads of an operator's arguments.  Its launch begins while the kernel before it may still be writing them, so
// none may take the read-only path (ld.global.nc, __ldg: for what nothing writes as long as the kernel runs, and
// free to move above the wait); as volatile statements they stay behind it.
__device__ __forceinline__ int32_t load_arg(const int32_t* p) {
  int32_t v;
  asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

__device__ __forceinline__ uint32_t load_arg(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

__device__ __forceinline__ float load_arg(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}

__device__ __forceinline__ uint2 load_arg(const uint2* p) {
  uint2 v;
  asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

__device__ __forceinline__ float4 load_arg(const float4* p) {
  float4 v;
  asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}

// The same of what is read once, not kept in L1; the second also keeps its place among the stores.
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ uint4 load_once_ordered(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// Four bytes to shared memory, zeros where there are none.
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src, bool valid) {
  const uint32_t bytes = valid ? 4u : 0u;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Four 8x8 matrices of 16-bit elements, each transposed: lane l receives, of matrix i, rows
// 2 (l % 4) and 2 (l % 4) + 1 of column l / 4 in r[i].
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// cap tanh(x) from one exponential: off by 2^-22 of the cap, infinities in it.
__device__ __forceinline__ float capped(float x, float cap) {
  float e, rate;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * 2.8853900817779268f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rate) : "f"(e + 1.0f));
  return fmaf(-2.0f * cap, rate, cap);
}

// cap tanh(x) and cap tanh(y) for |x|, |y| up to kTanhBound, by an odd polynomial with coefficients fitted to the least
// largest error there: off by 2^-23 of themselves and FP32's roundings, where the form above is off by 2^-22 of the cap; and
// without its two operations of the 4-lane unit, of a score's three.
constexpr float kTanhBound = 0.75f;
__device__ __forceinline__ void capped_pair(float& x, float& y, float cap) {
  asm("{\n .reg .b64 t, w, p, c;\n mov.b64 t, {%0, %1};\n mul.rn.f32x2 w, t, t;\n"
      " mov.b64 p, {%8, %8};\n mov.b64 c, {%7, %7};\n fma.rn.f32x2 p, p, w, c;\n mov.b64 c, {%6, %6};\n fma.rn.f32x2 p, p, w, c;\n"
      " mov.b64 c, {%5, %5};\n fma.rn.f32x2 p, p, w, c;\n mov.b64 c, {%4, %4};\n fma.rn.f32x2 p, p, w, c;\n"
      " mov.b64 c, {%3, %3};\n fma.rn.f32x2 p, p, w, c;\n mul.rn.f32x2 p, p, t;\n mov.b64 c, {%2, %2};\n mul.rn.f32x2 p, p, c;\n"
      " mov.b64 {%0, %1}, p;\n}"
      : "+f"(x), "+f"(y)
      : "f"(cap), "f"(0.99999983f), "f"(-0.33332471f), "f"(0.13320579f), "f"(-0.05314925f), "f"(0.01923722f), "f"(-0.00449344f));
}

// Two scores of one token times over_cap, capped by the form that fits them (so that no other token changes their bits).
__device__ __forceinline__ void cap_pair(float& x, float& y, float over_cap, float cap) {
  x *= over_cap, y *= over_cap;
  if (fmaxf(fabsf(x), fabsf(y)) <= kTanhBound) {
    capped_pair(x, y, cap);
  } else {
    x = capped(x, cap), y = capped(y, cap);
  }
}

}  // namespace chord
