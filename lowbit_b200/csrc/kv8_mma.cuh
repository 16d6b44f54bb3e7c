// Warp-level tensor-core pieces of the paged 8-bit attention kernels: codes to
// fp16, mma.sync with fp32 accumulators, 8x8 transposes, exp2.
#pragma once

#include "kv8.cuh"

namespace lbc {
namespace kv8 {

// four int8 codes -> two fp16 pairs (bytes 0,1 and 2,3), exactly: with the sign
// bit flipped a byte is code + 128, and 0x64 above it makes the half 1152 + code
__device__ __forceinline__ uint32_t half_pair(uint32_t biased, uint32_t sel) {
  uint32_t h;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(h) : "r"(prmt(biased, 0x64646464u, sel)), "r"(0x64806480u));
  return h;
}
__device__ __forceinline__ uint32_t half_lo(uint32_t biased) { return half_pair(biased, 0x4140); }
__device__ __forceinline__ uint32_t half_hi(uint32_t biased) { return half_pair(biased, 0x4342); }

// D[16,8] += A[16,16] B[16,8], fp16 in, fp32 accumulators
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// transpose of an 8x8 matrix of 16-bit elements held two a lane
__device__ __forceinline__ uint32_t transpose8(uint32_t r) {
  uint32_t o;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(o) : "r"(r));
  return o;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// two fp32 values in a register pair, and arithmetic on both at once
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ void split(uint64_t p, uint32_t &a, uint32_t &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  uint32_t h;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(b), "f"(a));
  return h;
}
// the rests a - fp16(a), b - fp16(b) of a packed pair
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t hi) {
  const float h0 = __half2float(__ushort_as_half((unsigned short)hi));
  const float h1 = __half2float(__ushort_as_half((unsigned short)(hi >> 16)));
  return pack_half(a - h0, b - h1);
}

// a power of two that brings |x| <= amax to at most 2^14 (its top to 2^13 and
// more), so that two fp16 pieces hold 22 bits of everything down to 2^-16 of
// the largest; NaN for non-finite rows: an infinite query makes every score
// infinite or NaN, so a row that sees anything is NaN (scores of -inf alone would
// look like a row that sees nothing)
__device__ __forceinline__ float fp16_range(float amax) {
  const int e = (int)(__float_as_uint(amax) >> 23) & 255;
  if (e == 255) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((uint32_t)(min(13 + 127 - e, 126) + 127) << 23);
}

// 16 bytes from global to shared memory, asynchronously
__device__ __forceinline__ void copy_async16(uint32_t dst, const int8_t *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void shared_words(uint32_t src, uint32_t *w) {
  if constexpr (BYTES == 16)
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(src) : "memory");
  else if constexpr (BYTES == 8)
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(src) : "memory");
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(src) : "memory");
}

}  // namespace kv8
}  // namespace lbc
