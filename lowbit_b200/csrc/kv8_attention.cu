// Causal grouped-query attention over the paged 8-bit KV cache
// (include/lowbit_b200.h: lbc_kv8_attention).
#include <cstdio>

#include "kernels.h"
#include "kv8.cuh"

namespace lbc {
namespace kv8 {
namespace {

constexpr int WARPS = 8;

struct AttnArgs {
  Pool c;
  Rows r;
  const void *q;
  long long ld;
  void *out;
  int H, window;
  float scale_log2;  // scale * log2(e)
};

// One CTA per row and head; warp w takes keys first + w, first + w + 8, ...
// with a running maximum and sum, lane l the elements l, l + 32, ...
template <typename T, int D>
__global__ void __launch_bounds__(WARPS * 32) attention_kernel(AttnArgs a) {
  constexpr int E = D / 32;
  __shared__ float sm[WARPS], sl[WARPS], so[WARPS][D];
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int r0, n;
  const int b = row_seq(a.r, row);
  seq_rows(a.r, b, r0, n);
  if (row < r0 || row >= r0 + n) return;
  int p = a.r.pos[b] + row - r0;
  if (p >= a.r.width << a.c.lg_page) {  // past the table: no keys
    set_status(a.r.status, LBC_ERR_PAGE);
    p = -1;
  }
  const int kvh = h / (a.H / a.c.KV);
  const int first = a.window > 0 ? max(0, p - a.window + 1) : 0;
  const T *q = static_cast<const T *>(a.q) + row * a.ld + (size_t)h * D;
  float qv[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qv[e] = to_f<T>(q[lane + 32 * e]);
    acc[e] = 0.f;
  }
  for (int j = first + warp; j <= p; j += WARPS) {
    const int id = page_id(a.c, a.r, b, j >> a.c.lg_page);
    if (id < 0) continue;
    const size_t at = id * a.c.page_stride + ((size_t)kvh * a.c.page + (j & (a.c.page - 1))) * D;
    const float ks = pow2_e8m0(a.c.k_exp[id * a.c.exp_stride + kvh]);
    const float vs = pow2_e8m0(a.c.v_exp[id * a.c.exp_stride + kvh]);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(qv[e], (float)a.c.k[at + lane + 32 * e], s);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s = s * ks * a.scale_log2;
    const float mn = fmaxf(m, s), f = exp2f(m - mn), w = exp2f(s - mn);
    l = fmaf(l, f, w);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(acc[e], f, w * vs * (float)a.c.v[at + lane + 32 * e]);
    m = mn;
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][lane + 32 * e] = acc[e];
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += WARPS * 32) {
    float mx = -INFINITY, den = 0.f, num = 0.f;
    for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, sm[w]);
    for (int w = 0; w < WARPS; ++w) {
      const float f = sm[w] == -INFINITY ? (sl[w] == 0.f ? 0.f : sl[w]) : exp2f(sm[w] - mx);  // a warp without keys adds nothing
      den = fmaf(sl[w], f, den);
      num = fmaf(so[w][d], f, num);
    }
    static_cast<T *>(a.out)[((size_t)row * a.H + h) * D + d] = from_f<T>(den == 0.f ? 0.f : num / den);
  }
}

template <typename T>
void launch(const AttnArgs &a, cudaStream_t st) {
  const dim3 grid(a.r.N, a.H);
  if (a.c.D == 32) attention_kernel<T, 32><<<grid, WARPS * 32, 0, st>>>(a);
  else if (a.c.D == 64) attention_kernel<T, 64><<<grid, WARPS * 32, 0, st>>>(a);
  else attention_kernel<T, 128><<<grid, WARPS * 32, 0, st>>>(a);
}

}  // namespace
}  // namespace kv8
}  // namespace lbc

using namespace lbc;
using namespace lbc::kv8;

extern "C" {

size_t lbc_kv8_attention_workspace(const lbc_kv8 *c, int dtype, int table_width, int B, int N, int max_tokens, int H,
                                   int window) {
  return 0;
}

int lbc_kv8_attention(const lbc_kv8 *c, int dtype, const void *q, long long ld, const int32_t *table, int table_width,
                      const int32_t *pos, const int32_t *starts, int B, int N, int max_tokens, int H, int window,
                      float scale, void *out, void *workspace, size_t workspace_bytes, void *stream) {
  AttnArgs a;
  int *status = nullptr, sms = 0;
  if (int rc = check_pool(c, a.c)) return rc;
  if (int rc = device_ready(&status, &sms)) return rc;
  if (int rc = check_rows(a.c, table, table_width, pos, starts, B, N, max_tokens, status, a.r)) return rc;
  if (dtype < LBC_F32 || dtype > LBC_F16) return refuse("kv8_attention: dtype must be fp32, bf16 or fp16");
  if (H <= 0 || H % a.c.KV || H > 65535) return refuse("kv8_attention: H must be a multiple of the KV heads");
  if (N == 0) return 0;
  if (!q || !out) return refuse("kv8_attention: NULL argument");
  if (ld < (long long)H * a.c.D || ld * (dtype == LBC_F32 ? 4 : 2) % 16) return refuse("kv8_attention: bad row stride");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15)
    return refuse("kv8_attention: q and out must be 16-byte aligned");
  a.q = q; a.ld = ld; a.out = out; a.H = H; a.window = window;
  a.scale_log2 = scale * 1.4426950408889634f;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == LBC_F32) launch<float>(a, st);
  else if (dtype == LBC_BF16) launch<__nv_bfloat16>(a, st);
  else launch<__half>(a, st);
  return launched("kv8_attention");
}

}  // extern "C"
