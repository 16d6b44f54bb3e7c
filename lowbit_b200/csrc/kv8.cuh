// Paged 8-bit KV cache: the pool's layout and the row / page lookups its
// kernels share. Layout and conventions: include/lowbit_b200.h (lbc_kv8).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace lbc {
namespace kv8 {

struct Pool {
  int8_t *k, *v;
  uint8_t *k_exp, *v_exp;
  long long page_stride, exp_stride;  // bytes from page to page (64-bit: pools pass 2^31 bytes)
  int pages, page, lg_page;           // page = 1 << lg_page tokens
  int KV, D;
};

// the sequences of one call
struct Rows {
  const int32_t *table, *pos, *starts;
  int width, B, N, most;  // table width (pages), sequences, rows; max_tokens (without starts: the rows of each)
  int *status;
};

// rows [r0, r0 + n) of sequence b; a sequence whose rows do not fit the
// call's limits keeps the rows that do, and the status word says so
__device__ __forceinline__ void seq_rows(const Rows &r, int b, int &r0, int &n) {
  if (!r.starts) {
    n = r.most;
    r0 = b * n;
    return;
  }
  const int lo = r.starts[b], hi = r.starts[b + 1];
  r0 = min(max(lo, 0), r.N);
  n = min(max(hi, r0), r.N) - r0;
  if (lo < 0 || hi < lo || hi > r.N || n > r.most) {
    set_status(r.status, LBC_ERR_PAGE);
    n = min(n, r.most);
  }
}

// id of the page that holds positions [o * page, (o + 1) * page) of sequence
// b, or -1 (recorded) when the table or the pool has no such page
__device__ __forceinline__ int page_id(const Pool &c, const Rows &r, int b, int o) {
  int id = -1;
  if (o >= 0 && o < r.width) id = r.table[(size_t)b * r.width + o];
  if (id < 0 || id >= c.pages) {
    set_status(r.status, LBC_ERR_PAGE);
    return -1;
  }
  return id;
}

// 2^(e - 127) from the float's bits; e = 0 is the subnormal 2^-127, 255 NaN
__device__ __forceinline__ float pow2_e8m0(int e) {
  return __uint_as_float(e == 255 ? 0x7fc00000u : e == 0 ? 0x00400000u : (uint32_t)e << 23);
}

// 2^(127 - e), e <= 254: every value is a normal float or, at e = 254, the subnormal 2^-127
__device__ __forceinline__ float pow2_inverse(int e) {
  return __uint_as_float(e == 254 ? 0x00400000u : (uint32_t)(254 - e) << 23);
}

// the smallest e >= 0 with amax <= 127 * 2^(e - 127); 255 for a non-finite amax.
// 127 = 1.984375 * 2^6: with amax = 1.f * 2^x, e - 127 is x - 6, one more when
// 1.f is above 1.984375. The exponent field is x + 127; below 6 the result is 0
// (which covers zero and subnormal amax).
__device__ __forceinline__ int scale_byte(float amax) {
  const uint32_t u = __float_as_uint(amax) & 0x7fffffffu;
  const int x = (int)(u >> 23);
  if (x == 255) return 255;
  return max(0, x - 6 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0));
}

// ------------------------------------------------------------ element types
template <typename T>
constexpr bool is_bf16 = false;
template <>
constexpr bool is_bf16<__nv_bfloat16> = true;
template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// four elements (16-byte aligned fp32, 8-byte aligned 16-bit types)
template <typename T>
__device__ __forceinline__ void load4(const T *p, float (&x)[4]) {
  if constexpr (sizeof(T) == 4) {
    const float4 v = *reinterpret_cast<const float4 *>(p);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else {
    union { uint2 u; T t[4]; } v;
    v.u = *reinterpret_cast<const uint2 *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = to_f<T>(v.t[i]);
  }
}
template <typename T>
__device__ __forceinline__ void store4(T *p, const float (&x)[4]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    union { uint2 u; T t[4]; } v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v.t[i] = from_f<T>(x[i]);
    *reinterpret_cast<uint2 *>(p) = v.u;
  }
}

// The kernels here are launched to start while the kernel before them in the
// stream finishes (programmatic stream serialisation). Every thread calls this
// before its first access to global memory: it returns when that kernel, and
// with it everything before, is over. (Global data is read with plain loads: a
// non-coherent one may be moved up.)
__device__ __forceinline__ void after_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets the kernel after start, to wait in turn. Short kernels do so at once
// (calls in a row: one token 8.7 -> 7.1 us, 16 sequences 13.8 -> 11.8); kernels
// that fill the GPU for long do not (64 sequences to 8192 tokens: 121 -> 150 us,
// the waiting blocks take the places of the next wave's).
__device__ __forceinline__ void next_kernel_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
void launch_chained(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, int cluster, cudaStream_t st, const A &...args) {
  cudaLaunchAttribute at[2] = {};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
}

// host: pool and row arguments checked and converted; 0 or LBC_ERR_SHAPE
int check_pool(const lbc_kv8 *c, Pool &out);
int check_rows(const Pool &c, const int32_t *table, int width, const int32_t *pos, const int32_t *starts, int B, int N,
               int most, int *status, Rows &out);

// records `why` and returns LBC_ERR_SHAPE
int refuse(const char *why);
// 0, or LBC_ERR_CUDA with the text of the launch error recorded
int launched(const char *what);

}  // namespace kv8
}  // namespace lbc
