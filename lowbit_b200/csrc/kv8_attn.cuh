// What the two attention kernels over the paged 8-bit KV cache share: the
// call's arguments and the geometry of a sequence's rows.
#pragma once

#include "kv8.cuh"
#include "kv8_mma.cuh"

namespace lbc {
namespace kv8 {

constexpr float LOWEST = -3e38f;  // M before any visible token
// Both kernels add block j's weights to l with 2^(f - b_j), f the largest value
// exponent looked up so far. That, and a weight that underflows while its share of
// l does not, is sound while the exponents looked up together lie within FAR and
// f grows by at most RISE after that (l <= 2^(15 + FAR + RISE) a token; a lost
// weight is below 2^-50 of l). Where they lie farther apart, the rows are computed
// by far_row. Blocks of exponent 0 whose codes are all 0 (a cache that was not
// filled) are left out of that: their codes do not matter, and their l counts with
// f - FAR, or, where f was 0 so far, follows f by way of M.
constexpr int FAR = 60, RISE = 30;

// fp16 pieces of queries and of weights: fp32 needs 22 bits of both; bf16 and
// fp16 queries are exact in one; fp16 outputs (11 bits) would show weights
// rounded to 11 bits (error 1.5 times the output's own). bf16 outputs round 8 times
// more coarsely: one piece makes their error 1.69e-3 -> 1.71e-3 (64 sequences to 8192
// tokens), in last places
template <typename T>
constexpr int QUERY_PIECES = sizeof(T) == 4 ? 2 : 1;
template <typename T>
constexpr int WEIGHT_PIECES = is_bf16<T> ? 1 : 2;

struct AttnArgs {
  Pool c;
  Rows r;
  const void *q;
  long long ld;
  void *out;
  int H, G, window;
  float scale_log2;  // scale * log2(e)
  int tiles;         // row tiles a sequence can have
  int split;         // 0: a cluster an item
  int2 *desc;        // [B][tiles][KV] first and last CTA of an item
  float *part;       // [grid][2] records: O [8 NQ][D], then M, l, f [8 NQ] each
  float *total;      // 16-bit calls over many tokens: a place for each thread's O so far (fold_sums); else null
};

// Tensor cores add to a running sum with truncation, so O drifts towards 0 with the
// number of tokens. fp32 calls add each step's O to a sum rounded to nearest. 16-bit
// outputs show it later: by 6.6e-9 a token in the prompt kernel with fp16's two weight
// pieces (8.7e-4 at 131072 tokens, the output's own rounding 2.2e-4), 4.6e-9 with
// bf16's one (6.0e-4, 1.0e-3); 2e-9 in the few-row kernel, whose four warps share
// the tokens. Where a row can see more than FOLD tokens (fp16: an eighth of the
// output's half ulp), or 16 times as many (bf16: a sixth), O is added to a total in
// the workspace each FOLD tokens and begun anew (131072 tokens then: 6e-5).
constexpr int FOLD = 8192;
inline bool fold_sums(int dtype, long long tokens) { return dtype != LBC_F32 && tokens > (dtype == LBC_F16 ? FOLD : 16 * FOLD); }

// sequence b: its rows, first position, units of UNIT tokens from the u0-th on,
// tiles of ROWS rows
struct Seq {
  int r0, n, p0, u0, units, tiles;
};
template <int UNIT, int ROWS>
__device__ __forceinline__ Seq seq_of(const AttnArgs &a, int b) {
  Seq s;
  seq_rows(a.r, b, s.r0, s.n);
  s.p0 = a.r.pos[b];
  const long long cap = (long long)a.r.width << a.c.lg_page;
  long long last = (long long)s.p0 + s.n - 1;
  if (s.n > 0 && last >= cap) {  // rows past the table see nothing
    set_status(a.r.status, LBC_ERR_PAGE);
    last = cap - 1;
  }
  int first = 0;
  if (a.window > 0) first = max(0, max(s.p0, 0) - a.window + 1);
  s.u0 = first / UNIT;
  s.units = s.n > 0 && last >= first ? (int)last / UNIT - s.u0 + 1 : 0;
  s.tiles = (s.n * a.G + ROWS - 1) / ROWS;
  return s;
}

// position of row `rho` (token rho / G) of a sequence, -1 for rows that see
// nothing; the rows that fill up the last tile (never stored) copy the last one
__device__ __forceinline__ int row_pos(const AttnArgs &a, const Seq &s, int rho) {
  const long long p = (long long)s.p0 + min(rho, s.n * a.G - 1) / a.G;
  return p >= ((long long)a.r.width << a.c.lg_page) ? -1 : (int)p;
}

// M for the largest t: `head` below it, rounded up; t itself where floats are too
// sparse for that (from 2^25 on `head` rounds to more than fp16 weights allow)
__device__ __forceinline__ float reference(float t, float head, float slack) {
  const float m = ceilf(t) - head;
  return t - m > slack ? t : m;
}

// One row over the tokens [j0, j1) by one warp, for value scales of any spread: in
// fp32 with the values themselves, o = 2^-lift sum 2^(z_j - m) v_j and l = sum
// 2^(z_j - m), m the largest z_j rounded up. A lane holds D / 32 elements. Not
// fast, and seldom run: a token at a time, with few registers, so that the
// kernels around it keep theirs.
template <typename T, int D>
__device__ __forceinline__ void far_row(const AttnArgs &a, int b, int kvh, const T *q, int p, int j0, int j1, int lift, int lane,
                                        float &m, float &l, float (&o)[D / 32]) {
  constexpr int E = D / 32;  // elements a lane
  const int lo = max(j0, a.window > 0 ? max(0, p - a.window + 1) : 0), hi = min(j1, p + 1);
  float x[E], amax = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    x[i] = to_f<T>(q[lane * E + i]);
    amax = x[i] == x[i] ? fmaxf(amax, fabsf(x[i])) : INFINITY;
  }
#pragma unroll
  for (int d = 16; d >= 1; d /= 2) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
  const float up = fp16_range(amax), back = a.scale_log2 / up, down = lift ? ex2(-(float)lift) : 1.f;
  m = LOWEST;
  l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    x[i] *= up;
    o[i] = 0.f;
  }
#pragma unroll 1
  for (int j = lo; j < hi; ++j) {
    const int id = a.r.table[(size_t)b * a.r.width + (j >> a.c.lg_page)];
    if ((unsigned)id >= (unsigned)a.c.pages) continue;
    const long long off = id * a.c.page_stride + ((long long)kvh * a.c.page + (j & (a.c.page - 1))) * D + lane * E;
    const long long at = id * a.c.exp_stride + kvh;
    float z = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) z = fmaf(x[i], (float)a.c.k[off + i], z);
#pragma unroll
    for (int d = 16; d >= 1; d /= 2) z += __shfl_xor_sync(0xffffffffu, z, d);
    z *= back * pow2_e8m0(a.c.k_exp[at]);
    const float to = fmaxf(m, ceilf(z)), f = ex2(m - to), w = ex2(z - to), value = pow2_e8m0(a.c.v_exp[at]) * down;
    m = to;
    l = fmaf(l, f, w);
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = fmaf(w, (float)a.c.v[off + i] * value, o[i] * f);
  }
}

// far_row's `lift` for the tokens [j0, j1) of sequence b: 20 where sums of the largest values could pass fp32's range
__device__ __forceinline__ int far_lift(const AttnArgs &a, int b, int kvh, int j0, int j1, int lane) {
  int top = 0;
  for (int i = (j0 >> a.c.lg_page) + lane; i < a.r.width && i <= (j1 - 1) >> a.c.lg_page; i += 32) {
    const int id = a.r.table[(size_t)b * a.r.width + i];
    const int ev = (unsigned)id < (unsigned)a.c.pages ? a.c.v_exp[id * a.c.exp_stride + kvh] : 255;
    if (ev != 255) top = max(top, ev);
  }
  return __any_sync(0xffffffffu, top > 220) ? 20 : 0;
}

// whether a 16-byte piece of block (page id, head kvh)'s value codes is not 0: of those that this thread, one of `step`, takes
__device__ __forceinline__ bool has_value(const AttnArgs &a, int id, int kvh, int thread, int step) {
  const int n = a.c.page * a.c.D / 16;
  const uint4 *p = reinterpret_cast<const uint4 *>(a.c.v + id * a.c.page_stride + (long long)kvh * a.c.page * a.c.D);
  uint32_t any = 0;
#pragma unroll 4
  for (int i = thread; i < n; i += step) {
    const uint4 v = p[i];
    any |= v.x | v.y | v.z | v.w;
  }
  return any != 0;
}

// y 2^x for a whole number x, in two steps, since 2^x alone may be too small for fp32
__device__ __forceinline__ float times_pow2(float y, float x) {
  const float h = truncf(0.5f * x);
  return y * ex2(h) * ex2(x - h);
}

// prompt chunks (kv8_prompt.cu), and the rows that one of its CTAs takes
int prompt_rows(int dtype, int D);
// floats of `total` a row of the prompt kernel needs: its O and its M
constexpr int total_row(int D) { return D + 4; }
void launch_prompt(const AttnArgs &a, int dtype, cudaStream_t st);

}  // namespace kv8
}  // namespace lbc
