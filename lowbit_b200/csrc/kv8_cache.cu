// Paged 8-bit KV cache: append (bias, position rotation, quantisation into the
// pages) and read-back. Layout and conventions: include/lowbit_b200.h (lbc_kv8).
//
// A block (the tokens of one page and head) has one owner CTA per call, so its
// exponent and codes are written without atomics and do not depend on the
// order in which CTAs run. Products and sums of the rotation are rounded
// separately (as lbc_qkv_rope does).
#include <algorithm>
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
  o.width = width; o.B = B; o.N = N; o.most = starts ? most : N / B;
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

constexpr int THREADS = 256, APPEND = 128;  // of the read and append kernels

__device__ __forceinline__ float block_max(float v, float *red) {
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, v, s);
    v = (v != v || o != o) ? __uint_as_float(0x7fc00000u) : fmaxf(v, o);
  }
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float m = red[0];
  for (int i = 1; i < (int)blockDim.x / 32; ++i) m = (m != m || red[i] != red[i]) ? __uint_as_float(0x7fc00000u) : fmaxf(m, red[i]);
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

template <typename T>
constexpr int VEC = 16 / (int)sizeof(T);  // elements of a 16-byte load

template <typename T>
__device__ __forceinline__ void load16(const T *p, float (&x)[VEC<T>]) {
  const uint4 u = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      x[i] = __uint_as_float(w[i]);
    } else {
      const ushort2 h = make_ushort2((unsigned short)w[i], (unsigned short)(w[i] >> 16));
      x[2 * i] = to_f<T>(reinterpret_cast<const T &>(h.x));
      x[2 * i + 1] = to_f<T>(reinterpret_cast<const T &>(h.y));
    }
  }
}
template <typename T>
__device__ __forceinline__ void store16(T *p, const float (&x)[VEC<T>]) {
  union {
    uint4 u;
    T t[VEC<T>];
  } v;
#pragma unroll
  for (int i = 0; i < VEC<T>; ++i) v.t[i] = from_f<T>(x[i]);
  *reinterpret_cast<uint4 *>(p) = v.u;
}

// V consecutive fp32 values of a table or bias (bias may lie at any float)
template <int V>
__device__ __forceinline__ void load_row(const float *p, float (&x)[V], bool aligned) {
  if (aligned) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 v = *reinterpret_cast<const float4 *>(p + i);
      x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = p[i];
  }
}

// elements [d, d + V) and [d + D/2, d + D/2 + V) of head `head` of a row, bias added
template <typename T, int D>
__device__ __forceinline__ void load_pair(const AppendArgs &a, int row, int head, int d, float (&x1)[VEC<T>], float (&x2)[VEC<T>]) {
  constexpr int V = VEC<T>;
  const int col = head * D + d;
  const T *src = static_cast<const T *>(a.qkv) + row * a.ld + col;
  load16<T>(src, x1);
  load16<T>(src + D / 2, x2);
  if (a.bias) {
    float b1[V], b2[V];
    const bool al = (reinterpret_cast<uintptr_t>(a.bias) & 15) == 0;
    load_row<V>(a.bias + col, b1, al);
    load_row<V>(a.bias + col + D / 2, b2, al);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x1[i] = __fadd_rn(x1[i], b1[i]);
      x2[i] = __fadd_rn(x2[i], b2[i]);
    }
  }
}

// rotate-half by the angles whose cosines and sines are c and s
template <int V>
__device__ __forceinline__ void turn(float (&x1)[V], float (&x2)[V], const float (&c)[V], const float (&s)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float o1 = __fsub_rn(__fmul_rn(x1[i], c[i]), __fmul_rn(x2[i], s[i]));
    const float o2 = __fadd_rn(__fmul_rn(x2[i], c[i]), __fmul_rn(x1[i], s[i]));
    x1[i] = o1;
    x2[i] = o2;
  }
}

template <int V>
__device__ __forceinline__ void store_codes(int8_t *dst, const float (&x)[V], float f, float top) {
  uint32_t w[V / 4];
#pragma unroll
  for (int i = 0; i < V / 4; ++i) w[i] = pack4({x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]}, f, top);
  if constexpr (V == 8) *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t *>(dst) = w[0];
}

// the sequence that owns row `row`, 32 of them compared at a time by the warp
__device__ __forceinline__ int warp_row_seq(const Rows &r, int row) {
  if (!r.starts) return row / r.most;
  int b = 0;
  for (int i = threadIdx.x & 31; i - (int)(threadIdx.x & 31) < r.B; i += 32) {
    const int k = __popc(__ballot_sync(0xffffffffu, i < r.B && r.starts[i + 1] <= row));
    b += k;
    if (k < 32) break;
  }
  return min(b, r.B - 1);
}

// Grid: first the query CTAs, one row a warp; then 2 * KV * slots * B CTAs, one
// block (keys or values of a page and head) each, whose work is shorter. A
// thread moves 16 bytes at a time; a block's rows are read twice, for the
// maximum and for the codes (the second time from L1: keeping them in registers
// costs the query CTAs their occupancy). 128 threads, so that more CTAs are in
// different phases of this (256: 37.1 us for 35.1; blocks first: 37.7), 64 when
// a sequence brings few rows.
// Bound by latency: one token 4.4 us, 64 sequences 6 us (launch, then table,
// rows, maximum, codes in turn); 6255 rows of 48 heads of 128, bf16, 35.1 us, 4.0
// TB/s of the 141 MB that it has to move.
template <typename T, int D>
__global__ void __launch_bounds__(APPEND, 8) append_kernel(AppendArgs a) {
  constexpr int V = VEC<T>, half = D / 2, per = half / V;  // per: threads a head and token
  __shared__ float red[APPEND / 32];
  after_previous_kernel();
  next_kernel_may_start();
  const int q_ctas = (a.r.N + blockDim.x / 32 - 1) / (blockDim.x / 32);
  int i = blockIdx.x;
  const int d = threadIdx.x % per * V;
  if (i < q_ctas) {  // queries, one row a warp: a lane keeps its angles for all its heads
    const int row = i * (blockDim.x / 32) + threadIdx.x / 32, lane = threadIdx.x & 31;
    if (row >= a.r.N) return;
    int r0, n;
    const int b = warp_row_seq(a.r, row);
    seq_rows(a.r, b, r0, n);
    if (row < r0 || row >= r0 + n) return;
    const long long p = (long long)a.r.pos[b] + row - r0;
    T *out = static_cast<T *>(a.q_out) + (size_t)row * a.H * D;
    if (p >= a.positions && lane == 0) set_status(a.r.status, LBC_ERR_PAGE);
    if (p < 0 || p >= a.positions) {
      float zero[V] = {};
      for (int head = lane / per; head < a.H; head += 32 / per) {
        store16<T>(out + head * D + d, zero);
        store16<T>(out + head * D + d + half, zero);
      }
      return;
    }
    float c[V], s[V];
    load_row<V>(a.cos_t + (size_t)p * half + d, c, true);
    load_row<V>(a.sin_t + (size_t)p * half + d, s, true);
#pragma unroll 4
    for (int head = lane / per; head < a.H; head += 32 / per) {
      float x1[V], x2[V];
      load_pair<T, D>(a, row, head, d, x1, x2);
      turn<V>(x1, x2, c, s);
      store16<T>(out + head * D + d, x1);
      store16<T>(out + head * D + d + half, x2);
    }
    return;
  }
  i -= q_ctas;
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
  const int head = a.H + (is_v ? a.c.KV : 0) + kvh, s0 = lo - (o << a.c.lg_page);
  const int step = blockDim.x / per;  // tokens apart
  const int t0 = threadIdx.x / per;
  // the thread's elements of token t of the block, k turned
  auto load = [&](int t, float (&x1)[V], float (&x2)[V]) {
    load_pair<T, D>(a, r0 + lo - pos + t, head, d, x1, x2);
    if (!is_v) {
      float c[V], s[V];
      load_row<V>(a.cos_t + (size_t)(lo + t) * half + d, c, true);
      load_row<V>(a.sin_t + (size_t)(lo + t) * half + d, s, true);
      turn<V>(x1, x2, c, s);
    }
  };
  float amax = 0.f;
#pragma unroll 2
  for (int t = t0; t < hi - lo; t += step) {
    float x1[V], x2[V];
    load(t, x1, x2);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      amax = fmaxf(amax, fmaxf(fabsf(x1[k]), fabsf(x2[k])));
      if (x1[k] != x1[k] || x2[k] != x2[k]) amax = INFINITY;
    }
  }
  if (id < 0) return;  // (asked only now: the rows are loaded meanwhile)
  int8_t *codes = (is_v ? a.c.v : a.c.k) + id * a.c.page_stride + (size_t)kvh * a.c.page * D;
  uint8_t *exp = (is_v ? a.c.v_exp : a.c.k_exp) + id * a.c.exp_stride + kvh;
  const int e_old = s0 == 0 ? 0 : *exp;
  amax = block_max(amax, red);  // its barrier also orders the read of *exp before the store below
  const int e_new = max(e_old, scale_byte(amax));
  const float top = top_code(e_new);
  if (e_new > e_old && s0 > 0) {
    const float f = pow2_e8m0(max(127 + e_old - e_new, 1));  // 2^(e_old - e_new); below 2^-8 every code is 0 anyway
    uint32_t *w = reinterpret_cast<uint32_t *>(codes);
    for (int e = threadIdx.x; e < s0 * D / 4; e += blockDim.x) {
      const uint32_t u = w[e];
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = (float)(int8_t)(u >> (8 * j));
      w[e] = pack4(x, f, top);
    }
  }
  const float inv = e_new == 255 ? 0.f : pow2_inverse(e_new);
#pragma unroll 2
  for (int t = t0; t < hi - lo; t += step) {
    float x1[V], x2[V];
    load(t, x1, x2);
    if (e_new == 255) {  // the block is NaN: its codes do not matter
#pragma unroll
      for (int k = 0; k < V; ++k) x1[k] = x2[k] = 0.f;
    }
    int8_t *dst = codes + (size_t)(s0 + t) * D + d;
    store_codes<V>(dst, x1, inv, top);
    store_codes<V>(dst + half, x2, inv, top);
  }
  if (threadIdx.x == 0) *exp = (uint8_t)e_new;
}

// A block (page of the list and head) is 2^lg pieces of VEC elements. A thread
// has FLY pieces of keys and of values in flight before its first store; every
// store is 16 bytes, in lane order. A CTA reads one block, or, where there are
// many that hold fewer pieces than its threads can fly, `take` of them (MANY):
// 97 MB of pages of 16 tokens, D = 64, 31.1 -> 17.1 us. Looking the block up for
// every piece costs large ones time (pages of 64, D = 128: 64 -> 73 us), and few
// ones latency (8.2 -> 10.2 us from an idle GPU), so both keep one block a CTA.
// Bound by HBM: 402 MB of pages of 64, D = 128, to bf16 in 64 us, 6.3 TB/s.
constexpr int FLY = 4;
template <typename T, bool MANY>
__global__ void __launch_bounds__(THREADS) read_kernel(Pool c, const int32_t *ids, unsigned blocks, int lg, int take, T *k_out, T *v_out,
                                                       int *status) {
  after_previous_kernel();
  next_kernel_may_start();
  constexpr int V = VEC<T>;
  struct Block {
    long long at;  // bytes to its codes (a page that does not exist: any)
    float f[2];
    bool ok;
  };
  auto look_up = [&](unsigned block, bool record) {
    const unsigned page = block / c.KV, kvh = block - page * c.KV;
    const int id = ids[page];
    Block y;
    y.ok = id >= 0 && id < c.pages;
    if (!y.ok && record) set_status(status, LBC_ERR_PAGE);
    y.at = y.ok ? id * c.page_stride + (long long)kvh * c.page * c.D : 0;
    const long long scale = y.ok ? id * c.exp_stride + kvh : 0;
    y.f[0] = y.ok ? pow2_e8m0(c.k_exp[scale]) : 0.f;
    y.f[1] = y.ok ? pow2_e8m0(c.v_exp[scale]) : 0.f;
    return y;
  };
  const unsigned first = blockIdx.x * take, n = (MANY ? min((unsigned)take, blocks - first) : 1u) << lg;
  Block y[MANY ? FLY : 1];
  if constexpr (!MANY) y[0] = look_up(first, threadIdx.x == 0);
  T *out[2] = {k_out + ((size_t)first << lg) * V, v_out + ((size_t)first << lg) * V};
  for (unsigned e0 = threadIdx.x; e0 < n; e0 += FLY * THREADS) {
    uint32_t w[2][FLY][V / 4];
    if constexpr (MANY) {
#pragma unroll
      for (int u = 0; u < FLY; ++u) {
        const unsigned e = e0 + u * THREADS;
        if (e < n) y[u] = look_up(first + (e >> lg), (e & ((1u << lg) - 1)) == 0);
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int u = 0; u < FLY; ++u) {
        const unsigned e = e0 + u * THREADS;
        const int8_t *src = (s ? c.v : c.k) + y[MANY ? u : 0].at + (MANY ? e & ((1u << lg) - 1) : e) * V;
        if (e < n) {
          if constexpr (V == 8) {
            const uint2 x = *reinterpret_cast<const uint2 *>(src);
            w[s][u][0] = x.x;
            w[s][u][1] = x.y;
          } else {
            w[s][u][0] = *reinterpret_cast<const uint32_t *>(src);
          }
        }
      }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int u = 0; u < FLY; ++u) {
        const unsigned e = e0 + u * THREADS;
        if (e < n) {
          const Block &z = y[MANY ? u : 0];
          float x[V];
#pragma unroll
          for (int j = 0; j < V; ++j) x[j] = z.ok ? __fmul_rn((float)(int8_t)(w[s][u][j / 4] >> (8 * (j % 4))), z.f[s]) : 0.f;
          store16<T>(out[s] + (size_t)e * V, x);
        }
      }
  }
}

template <typename T>
void launch_read(const Pool &c, const int32_t *ids, int n, void *k_out, void *v_out, int *status, int sms, cudaStream_t st) {
  const unsigned blocks = (unsigned)n * c.KV;
  int lg = 0;
  while (VEC<T> << lg < c.page * c.D) ++lg;
  const int take = blocks / 8 < (unsigned)sms ? 1 : std::max(1, FLY * THREADS >> lg);
  launch_chained(take > 1 ? read_kernel<T, true> : read_kernel<T, false>, dim3((blocks - 1) / take + 1), THREADS, 0, 1, st, c, ids,
                 blocks, lg, take, static_cast<T *>(k_out), static_cast<T *>(v_out), status);
}

template <typename T>
void launch_append(const AppendArgs &a, long long kv_ctas, cudaStream_t st) {
  // 2 to 16 threads a token: up to 4 tokens need no more than 64
  const unsigned threads = a.r.most <= 4 ? 64 : APPEND, ctas = (unsigned)(kv_ctas + (a.r.N + threads / 32 - 1) / (threads / 32));
  if (a.c.D == 32) launch_chained(append_kernel<T, 32>, dim3(ctas), threads, 0, 1, st, a);
  else if (a.c.D == 64) launch_chained(append_kernel<T, 64>, dim3(ctas), threads, 0, 1, st, a);
  else launch_chained(append_kernel<T, 128>, dim3(ctas), threads, 0, 1, st, a);
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
  const long long ctas = 2LL * a.c.KV * a.slots * B;
  if (ctas + N > 0x7fffffffLL) return refuse("kv8_append: too many rows");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == LBC_F32) launch_append<float>(a, ctas, st);
  else if (dtype == LBC_BF16) launch_append<__nv_bfloat16>(a, ctas, st);
  else launch_append<__half>(a, ctas, st);
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
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == LBC_F32) launch_read<float>(p, ids, n, k_out, v_out, status, sms, st);
  else if (dtype == LBC_BF16) launch_read<__nv_bfloat16>(p, ids, n, k_out, v_out, status, sms, st);
  else launch_read<__half>(p, ids, n, k_out, v_out, status, sms, st);
  return launched("kv8_read");
}

}  // extern "C"
