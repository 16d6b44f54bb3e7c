// Paged 8-bit KV cache: append (bias, position rotation, quantisation into the
// pages) and read-back. Layout and conventions: include/lowbit_b200.h (lbc_kv8).
//
// A block (the tokens of one page and head) has one owner CTA per call, so its
// exponent and codes are written without atomics and do not depend on the
// order in which CTAs run. Products and sums of the rotation are rounded
// separately (as lbc_qkv_rope does).
#include <cstdio>

#include "kernels.h"
#include "kv8.cuh"

namespace lbc {
namespace kv8 {

int check_pool(const lbc_kv8 *c, Pool &o) {
  const char *why = nullptr;
  if (!c || !c->k || !c->v || !c->k_exp || !c->v_exp) why = "kv8: NULL cache";
  else if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128) why = "kv8: page must be 16, 32, 64 or 128 tokens";
  else if (c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128) why = "kv8: head_dim must be 32, 64 or 128";
  else if (c->pages <= 0 || c->kv_heads <= 0 || c->kv_heads > 1024) why = "kv8: bad pool shape";
  else if (c->page_stride < (long long)c->kv_heads * c->page * c->head_dim || c->page_stride % 16 || c->exp_stride < c->kv_heads)
    why = "kv8: bad page stride";
  else if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) why = "kv8: pools must be 16-byte aligned";
  if (why) {
    set_last_error(why);
    return LBC_ERR_SHAPE;
  }
  o.k = c->k; o.v = c->v; o.k_exp = c->k_exp; o.v_exp = c->v_exp;
  o.page_stride = c->page_stride; o.exp_stride = c->exp_stride;
  o.pages = c->pages; o.page = c->page; o.KV = c->kv_heads; o.D = c->head_dim;
  o.lg_page = c->page == 16 ? 4 : c->page == 32 ? 5 : c->page == 64 ? 6 : 7;
  return 0;
}

int check_rows(const Pool &c, const int32_t *table, int width, const int32_t *pos, const int32_t *starts, int B, int N,
               int most, int *status, Rows &o) {
  const char *why = nullptr;
  if (B <= 0 || B > 65535 || N < 0 || most < 0 || most > N) why = "kv8: bad row counts";
  else if (!table || !pos) why = "kv8: NULL page table or positions";
  else if (width <= 0 || ((long long)width << c.lg_page) > 0x7fffffffLL - 256) why = "kv8: bad page table width";
  else if (!starts && (N % B || most < N / B)) why = "kv8: without starts, N must be B times at most max_tokens";
  if (why) {
    set_last_error(why);
    return LBC_ERR_SHAPE;
  }
  o.table = table; o.pos = pos; o.starts = starts;
  o.width = width; o.B = B; o.N = N; o.most = most;
  o.status = status;
  return 0;
}

int refuse(const char *why) {
  set_last_error(why);
  return LBC_ERR_SHAPE;
}

int launched(const char *what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return 0;
  char buf[256];
  snprintf(buf, sizeof buf, "%s: %s", what, cudaGetErrorString(e));
  set_last_error(buf);
  return LBC_ERR_CUDA;
}

namespace {

constexpr int THREADS = 256;

__device__ __forceinline__ float block_max(float v, float *red) {
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, v, s);
    v = (v != v || o != o) ? __uint_as_float(0x7fc00000u) : fmaxf(v, o);
  }
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float m = red[0];
#pragma unroll
  for (int i = 1; i < THREADS / 32; ++i) m = (m != m || red[i] != red[i]) ? __uint_as_float(0x7fc00000u) : fmaxf(m, red[i]);
  return m;
}

// the largest code of a block: 127, but 64 * 2^122 (e = 249, the largest finite
// inputs) is past the largest float, so that exponent's codes stop at 63
__device__ __forceinline__ float top_code(int e) { return e == 249 ? 63.f : 127.f; }

// four codes rne(x * f), at most `top` in magnitude
__device__ __forceinline__ uint32_t pack4(const float (&x)[4], float f, float top) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= (uint32_t)((int)fminf(fmaxf(rintf(__fmul_rn(x[i], f)), -top), top) & 0xff) << (8 * i);
  return w;
}

struct AppendArgs {
  Pool c;
  Rows r;
  const void *qkv;
  long long ld;
  const float *bias, *cos_t, *sin_t;
  int positions, H, slots;  // slots: pages a sequence's rows can touch
  void *q_out;
};

// elements [d, d + 4) and [d + D/2, d + D/2 + 4) of head `head` of a row, bias
// added and, where `rotate`, turned by the position's angle
template <typename T>
__device__ __forceinline__ void load_pair(const AppendArgs &a, int row, int head, int d, int p, bool rotate, float (&x1)[4],
                                          float (&x2)[4]) {
  const int D = a.c.D, half = D / 2, col = head * D + d;
  const T *src = static_cast<const T *>(a.qkv) + row * a.ld + col;
  load4<T>(src, x1);
  load4<T>(src + half, x2);
  if (a.bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x1[i] = __fadd_rn(x1[i], a.bias[col + i]);
      x2[i] = __fadd_rn(x2[i], a.bias[col + half + i]);
    }
  }
  if (rotate) {
    float c[4], s[4];
    load4<float>(a.cos_t + (size_t)p * half + d, c);
    load4<float>(a.sin_t + (size_t)p * half + d, s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float o1 = __fsub_rn(__fmul_rn(x1[i], c[i]), __fmul_rn(x2[i], s[i]));
      const float o2 = __fadd_rn(__fmul_rn(x2[i], c[i]), __fmul_rn(x1[i], s[i]));
      x1[i] = o1;
      x2[i] = o2;
    }
  }
}

// grid: first 2 * KV * slots * B CTAs, one block (keys or values of a page and
// head) each; then the query CTAs, one row each
template <typename T>
__global__ void __launch_bounds__(THREADS) append_kernel(AppendArgs a) {
  __shared__ float red[THREADS / 32];
  const int D = a.c.D, half = D / 2, per = half / 4;  // pairs of four per head and token
  const int kv_ctas = 2 * a.c.KV * a.slots * a.r.B;
  int i = blockIdx.x;
  if (i >= kv_ctas) {  // queries of one row
    const int row = i - kv_ctas;
    int r0, n;
    const int b = row_seq(a.r, row);
    seq_rows(a.r, b, r0, n);
    if (row < r0 || row >= r0 + n) return;
    const long long p = (long long)a.r.pos[b] + row - r0;
    T *out = static_cast<T *>(a.q_out) + (size_t)row * a.H * D;
    if (p >= a.positions && threadIdx.x == 0) set_status(a.r.status, LBC_ERR_PAGE);
    for (int e = threadIdx.x; e < a.H * per; e += THREADS) {
      const int head = e / per, d = (e % per) * 4;
      float x1[4] = {0.f, 0.f, 0.f, 0.f}, x2[4] = {0.f, 0.f, 0.f, 0.f};
      if (p >= 0 && p < a.positions) load_pair<T>(a, row, head, d, (int)p, true, x1, x2);
      store4<T>(out + head * D + d, x1);
      store4<T>(out + head * D + d + half, x2);
    }
    return;
  }
  const bool is_v = i & 1;
  i >>= 1;
  const int kvh = i % a.c.KV;
  i /= a.c.KV;
  const int slot = i % a.slots, b = i / a.slots;
  int r0, n;
  seq_rows(a.r, b, r0, n);
  const int pos = a.r.pos[b];
  // positions [lo, hi) of this block's page: rows at negative positions or past the rotation tables are left out
  const int first = max(pos, 0), last = (int)min((long long)pos + n, (long long)a.positions);
  const int o = (first >> a.c.lg_page) + slot;
  const int lo = max(first, o << a.c.lg_page), hi = min(last, (o + 1) << a.c.lg_page);
  if (lo >= hi) return;
  const int id = page_id(a.c, a.r, b, o);
  if (id < 0) return;
  int8_t *codes = (is_v ? a.c.v : a.c.k) + id * a.c.page_stride + (size_t)kvh * a.c.page * D;
  uint8_t *exp = (is_v ? a.c.v_exp : a.c.k_exp) + id * a.c.exp_stride + kvh;
  const int head = a.H + (is_v ? a.c.KV : 0) + kvh, s0 = lo - (o << a.c.lg_page);
  const int work = (hi - lo) * per;
  float amax = 0.f;
  for (int e = threadIdx.x; e < work; e += THREADS) {
    float x1[4], x2[4];
    const int t = e / per;
    load_pair<T>(a, r0 + lo - pos + t, head, (e % per) * 4, lo + t, !is_v, x1, x2);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float m = fmaxf(fabsf(x1[j]), fabsf(x2[j]));
      if (x1[j] != x1[j] || x2[j] != x2[j]) amax = __uint_as_float(0x7f800000u);
      else amax = fmaxf(amax, m);
    }
  }
  const int e_old = s0 == 0 ? 0 : *exp;
  amax = block_max(amax, red);  // its barrier also orders the read of *exp before the store below
  const int e_new = max(e_old, scale_byte(amax));
  const float top = top_code(e_new);
  if (e_new > e_old && s0 > 0) {
    const float f = pow2_e8m0(max(127 + e_old - e_new, 1));  // 2^(e_old - e_new); below 2^-8 every code is 0 anyway
    uint32_t *w = reinterpret_cast<uint32_t *>(codes);
    for (int e = threadIdx.x; e < s0 * D / 4; e += THREADS) {
      const uint32_t u = w[e];
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = (float)(int8_t)(u >> (8 * j));
      w[e] = pack4(x, f, top);
    }
  }
  const float inv = e_new == 255 ? 0.f : pow2_inverse(e_new);
  for (int e = threadIdx.x; e < work; e += THREADS) {
    float x1[4], x2[4];
    const int t = e / per, d = (e % per) * 4;
    load_pair<T>(a, r0 + lo - pos + t, head, d, lo + t, !is_v, x1, x2);
    uint32_t *dst = reinterpret_cast<uint32_t *>(codes + (size_t)(s0 + t) * D + d);
    dst[0] = e_new == 255 ? 0 : pack4(x1, inv, top);
    dst[half / 4] = e_new == 255 ? 0 : pack4(x2, inv, top);
  }
  if (threadIdx.x == 0) *exp = (uint8_t)e_new;
}

// one CTA per (page of the list, head), keys then values
template <typename T>
__global__ void __launch_bounds__(THREADS) read_kernel(Pool c, const int32_t *ids, T *k_out, T *v_out, int *status) {
  const int i = blockIdx.x / c.KV, kvh = blockIdx.x % c.KV, n4 = c.page * c.D / 4;
  const int id = ids[i];
  const bool ok = id >= 0 && id < c.pages;
  if (!ok && threadIdx.x == 0) set_status(status, LBC_ERR_PAGE);
  for (int s = 0; s < 2; ++s) {
    T *out = (s ? v_out : k_out) + (size_t)blockIdx.x * c.page * c.D;
    const size_t at = ok ? id * c.page_stride + (size_t)kvh * c.page * c.D : 0;
    const uint32_t *w = reinterpret_cast<const uint32_t *>((s ? c.v : c.k) + at);
    const float f = ok ? pow2_e8m0((s ? c.v_exp : c.k_exp)[id * c.exp_stride + kvh]) : 0.f;
    for (int e = threadIdx.x; e < n4; e += THREADS) {
      const uint32_t u = ok ? w[e] : 0;
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = __fmul_rn((float)(int8_t)(u >> (8 * j)), f);
      store4<T>(out + 4 * (size_t)e, x);
    }
  }
}

}  // namespace
}  // namespace kv8
}  // namespace lbc

using namespace lbc;
using namespace lbc::kv8;

extern "C" {

int lbc_kv8_append(const lbc_kv8 *c, int dtype, const void *qkv, long long ld, const float *bias, const float *cos_t,
                   const float *sin_t, int positions, const int32_t *table, int table_width, const int32_t *pos,
                   const int32_t *starts, int B, int N, int max_tokens, int H, void *q_out, void *stream) {
  AppendArgs a;
  int *status = nullptr, sms = 0;
  if (int rc = check_pool(c, a.c)) return rc;
  if (int rc = device_ready(&status, &sms)) return rc;
  if (int rc = check_rows(a.c, table, table_width, pos, starts, B, N, max_tokens, status, a.r)) return rc;
  if (dtype < LBC_F32 || dtype > LBC_F16) return refuse("kv8_append: dtype must be fp32, bf16 or fp16");
  const int es = dtype == LBC_F32 ? 4 : 2, D = a.c.D;
  if (H <= 0 || H % a.c.KV || H > 65536) return refuse("kv8_append: H must be a multiple of the KV heads");
  if (N == 0) return 0;
  if (!qkv || !q_out || !cos_t || !sin_t || positions <= 0) return refuse("kv8_append: NULL argument");
  if (ld < (long long)(H + 2 * a.c.KV) * D || ld * es % 16) return refuse("kv8_append: bad row stride");
  if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(cos_t) |
       reinterpret_cast<uintptr_t>(sin_t)) & 15)
    return refuse("kv8_append: qkv, q_out, cos and sin must be 16-byte aligned");
  a.qkv = qkv; a.ld = ld; a.bias = bias; a.cos_t = cos_t; a.sin_t = sin_t;
  a.positions = positions; a.H = H; a.q_out = q_out;
  a.slots = (max_tokens + a.c.page - 2) / a.c.page + 1;
  const long long ctas = 2LL * a.c.KV * a.slots * B + N;
  if (ctas > 0x7fffffffLL) return refuse("kv8_append: too many rows");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == LBC_F32) append_kernel<float><<<(unsigned)ctas, THREADS, 0, st>>>(a);
  else if (dtype == LBC_BF16) append_kernel<__nv_bfloat16><<<(unsigned)ctas, THREADS, 0, st>>>(a);
  else append_kernel<__half><<<(unsigned)ctas, THREADS, 0, st>>>(a);
  return launched("kv8_append");
}

int lbc_kv8_read(const lbc_kv8 *c, int dtype, const int32_t *ids, int n, void *k_out, void *v_out, void *stream) {
  Pool p;
  int *status = nullptr, sms = 0;
  if (int rc = check_pool(c, p)) return rc;
  if (int rc = device_ready(&status, &sms)) return rc;
  if (dtype < LBC_F32 || dtype > LBC_F16) return refuse("kv8_read: dtype must be fp32, bf16 or fp16");
  if (n < 0 || (long long)n * p.KV > 0x7fffffffLL) return refuse("kv8_read: bad page count");
  if (n == 0) return 0;
  if (!ids || !k_out || !v_out) return refuse("kv8_read: NULL argument");
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15)
    return refuse("kv8_read: outputs must be 16-byte aligned");
  const unsigned ctas = (unsigned)n * p.KV;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == LBC_F32)
    read_kernel<float><<<ctas, THREADS, 0, st>>>(p, ids, static_cast<float *>(k_out), static_cast<float *>(v_out), status);
  else if (dtype == LBC_BF16)
    read_kernel<__nv_bfloat16><<<ctas, THREADS, 0, st>>>(p, ids, static_cast<__nv_bfloat16 *>(k_out),
                                                         static_cast<__nv_bfloat16 *>(v_out), status);
  else
    read_kernel<__half><<<ctas, THREADS, 0, st>>>(p, ids, static_cast<__half *>(k_out), static_cast<__half *>(v_out), status);
  return launched("kv8_read");
}

}  // extern "C"
