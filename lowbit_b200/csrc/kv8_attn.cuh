// What the two attention kernels over the paged 8-bit KV cache share: the
// call's arguments and the geometry of a sequence's rows.
#pragma once

#include "kv8.cuh"
#include "kv8_mma.cuh"

namespace lbc {
namespace kv8 {

constexpr float LOWEST = -3e38f;  // M before any visible token
// blocks whose value scale is 2^60 below the largest count with 2^(f - 60): they
// only matter to l (an all-zero block has exponent 0)
constexpr int FAR = 60;

// fp16 pieces of queries and of weights: fp32 needs 22 bits of both; bf16 and
// fp16 queries are exact in one; fp16 outputs (11 bits) would show weights
// rounded to 11 bits (error 1.5 times the output's own), bf16 ones do not
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
};

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

// prompt chunks (kv8_prompt.cu), and the rows that one of its CTAs takes
int prompt_rows(int dtype, int D);
void launch_prompt(const AttnArgs &a, int dtype, cudaStream_t st);

}  // namespace kv8
}  // namespace lbc
