// Causal grouped-query attention over the paged 8-bit KV cache
// (include/lowbit_b200.h: lbc_kv8_attention): softmax(scale q.k) v with a
// running maximum, one pass over the codes.
//
// Scores and outputs are computed transposed on mma.sync m16n8k16: 16 tokens
// (scores) or 16 elements (outputs) by 8 query rows, so that few rows (one
// token's G = H / KV heads) fill the tile. int8 codes are exact in fp16;
// queries are scaled by a power of two per row into fp16's range (fp32 ones as
// two pieces, 22 bits), weights likewise (fp32 and fp16: two pieces; bf16: one).
// Contraction indices may be permuted freely, and are: a lane loads 16
// contiguous bytes of its token's key (or of four tokens' values) as operand
// registers. Codes reach shared memory by cp.async in whole rows (half rows
// cost twice the L2 traffic), 16-byte pieces permuted so that neither read
// meets a bank twice; every warp has its own ring, so warps keep several
// steps in flight and need no barriers.
//
// With z_j = log2(e) scale q.k_j the weights carry their block's value scale
// 2^b_j: t_j = z_j + b_j, M about max t_j - 14 the running reference,
//   O = sum_j 2^(t_j - M) code_j,  l = sum_j 2^(t_j - M) 2^(f - b_j),
//   out = 2^f O / l,  f = max b_j,
// so weights stay within fp16, and all rescaling is by powers of two (M is a
// whole number). f is the largest b looked up, seen by a row or not; where they
// lie more than 2^60 apart, rows are computed one by one (kv8_attn.cuh: far_row).
//
// Work: an item is (sequence, tile of 8 NQ rows, KV head); its visible tokens
// are cut into units of 64 (16 a warp). The units of all items form one line
// that is cut evenly over the grid, wherever lengths differ: a CTA runs
// through the ends of items and whole ones; cut items leave partial
// (O, M, l, f) records that a second kernel joins in order (no atomics). When
// all items' longest possible ranges fit one wave of the grid anyway (few
// sequences, short tables), a cluster of up to 8 CTAs takes an item instead and
// joins its sums through distributed shared memory: one launch, no workspace.
//
// Bounds: long batches HBM (bf16, 32 heads, 8 KV heads of 128: 64 sequences to
// 8192 tokens 120-131 us from GPU to GPU, 5.0-5.5 TB/s; one of 131071 58 us, 4.6
// TB/s, the rest is the pipelines' start and the join); short ones the chain of
// launch, page lookup and units (14 heads, 2 KV heads of 64, fp32: 510 tokens 6.4
// us, 16 sequences to 4096 11.4 us); tiles of 24 rows issue and tensor-core latency
// (16 sequences of 5 tokens, 32 heads, window 1024, fp16: 24-25.5 us).
#include <algorithm>
#include <cstdio>

#include "kernels.h"
#include "kv8_attn.cuh"

namespace lbc {
namespace kv8 {
namespace {

// CTAs an SM that the registers allow. bf16 tiles of 16 rows fit three times at
// D <= 64: 9 sequences to 64000 tokens, 8 KV heads, 116 -> 110 us (D = 64), 88 ->
// 79 (D = 32); 15 to 11600, 1 KV head, 16.6 -> 17.5. fp16's second weight piece
// leaves it at two (19.8 -> 20.3).
constexpr int resident(int dtype, int D, int nq) {
  return nq == 2 && D < 128 && dtype == LBC_BF16 ? 3 : nq > 1 ? 2 : dtype == LBC_F32 && D == 128 ? 3 : 4;
}
template <typename T>
constexpr int DTYPE = sizeof(T) == 4 ? LBC_F32 : is_bf16<T> ? LBC_BF16 : LBC_F16;
constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int WTOK = 16;            // tokens of a warp in a unit
constexpr int UNIT = WARPS * WTOK;
constexpr int META = 128;           // pages looked up at a time
// weights 2^(t - M) fill fp16's range: M is the maximum (rounded up) less 14,
// left alone while no weight passes 2^15. Two pieces then hold a weight to 22
// bits down to 2^-17 of the largest, one piece to 11 bits down to 2^-28.
constexpr float HEAD = 14.f, SLACK = 15.f;

struct Meta {
  long long off[META];  // bytes to the block's codes (a page that does not exist: to page 0's)
  float4 s[META];       // 2^(ek - 127), b = ev - 127, 2^(f - b), 1 if the page exists
  int f;                // largest value exponent so far (255 left out)
};

// Ring steps of a warp: more where they are smaller. Measured 2 / 3 / 4 / 6 at
// D = 64 (13 sequences to 39520 tokens): 75.7 / 67.8 / 67.9 / 71.9 us; 2 / 3 at
// D = 128 (64 to 8192): 122 / 130.
template <int D>
constexpr int STAGES = D == 128 ? 2 : D == 64 ? 3 : 4;

template <typename T, int D, int NQ>
struct Warp {
  static constexpr int QP = QUERY_PIECES<T>, WP = WEIGHT_PIECES<T>;
  static constexpr int KW = D / 16, VW = D / 32, MT = D / 16;
  uint32_t q[NQ][QP][KW][2];  // query operand
  float rowf[NQ][2];              // score = accumulator * rowf * 2^(ek - 127), in log2 units
  int p[NQ][2];                   // positions of the lane's rows 8 n + 2 t + i
  float m[NQ][2], l[NQ][2], o[NQ][MT][4];

  // first element of the four that lane t's word s of a key row holds
  __device__ static int key_dim(int t, int s) { return t * (D / 4) + 4 * s; }

  // the lane's query elements, row 8 n + g of the tile, four at a time as they lie in memory; taken up by start()
  struct Query {
    struct alignas(4 * sizeof(T)) Four {
      T e[4];
    } x[NQ][KW];
  };
  __device__ __forceinline__ void load_query(Query &y, const AttnArgs &a, const Seq &s, int tile, int kvh, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int rho = (tile * NQ + n) * 8 + g;
      if (rho < s.n * a.G) {
        const int tok = rho < a.G ? 0 : rho / a.G, h = rho - tok * a.G;  // (one token: no division)
        const T *src = static_cast<const T *>(a.q) + (s.r0 + tok) * a.ld + (size_t)(kvh * a.G + h) * D;
#pragma unroll
        for (int w = 0; w < KW; ++w) y.x[n][w] = *reinterpret_cast<const typename Query::Four *>(src + key_dim(t, w));
      } else {
#pragma unroll
        for (int w = 0; w < KW; ++w) y.x[n][w].e[0] = y.x[n][w].e[1] = y.x[n][w].e[2] = y.x[n][w].e[3] = from_f<T>(0.f);
      }
    }
  }
  __device__ __forceinline__ void start(const Query &y, const AttnArgs &a, const Seq &s, int tile, int lane) {
    const int t = lane & 3;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float amax = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = to_f<T>(y.x[n][w].e[i]);
          amax = x == x ? fmaxf(amax, fabsf(x)) : INFINITY;
        }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const float f = fp16_range(amax);
#pragma unroll
      for (int w = 0; w < KW; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float x0 = to_f<T>(y.x[n][w].e[2 * h]) * f, x1 = to_f<T>(y.x[n][w].e[2 * h + 1]) * f;
          q[n][0][w][h] = pack_half(x0, x1);
          if constexpr (QP == 2) q[n][1][w][h] = pack_rest(x0, x1, q[n][0][w][h]);
        }
      const float back = a.scale_log2 / f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        rowf[n][i] = __shfl_sync(0xffffffffu, back, (2 * t + i) * 4);
        p[n][i] = row_pos(a, s, (tile * NQ + n) * 8 + 2 * t + i);
        m[n][i] = LOWEST;
        l[n][i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }
  }

  // one ring step: 16 tokens' keys, then their values
  static constexpr int STEP = 32 * D;
  // byte offset of 16-byte piece c of row r: pieces change places within their 128-byte line
  __device__ static int place(int r, int c) {
    constexpr int RL = 128 / D, PR = D / 16;  // rows a line, pieces a row
    return (r / RL) * 128 + (((r % RL * PR + c) ^ (D == 128 ? r & 7 : D == 64 ? (r >> 1 & 3) << 1 : (r >> 2 & 1) << 1)) << 4);
  }
  __device__ __forceinline__ void fetch(const AttnArgs &a, uint32_t step, long long off, int lane) {
    constexpr int PR = D / 16, RI = 32 / PR;  // rows an instruction copies
    const int8_t *k = a.c.k + off + lane * 16, *v = a.c.v + off + lane * 16;
#pragma unroll
    for (int i = 0; i < 16 / RI; ++i) {
      const int at = place(lane / PR + i * RI, lane % PR);
      copy_async16(step + at, k + i * 512);
      copy_async16(step + 16 * D + at, v + i * 512);
    }
  }

  // scores of the step's 16 tokens, in units of rowf * 2^(ek - 127)
  __device__ __forceinline__ void scores(float (&z)[NQ][4], uint32_t step, int lane) {
    uint32_t k[2][KW];
#pragma unroll
    for (int n = 0; n < NQ; ++n) z[n][0] = z[n][1] = z[n][2] = z[n][3] = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = (lane >> 2) + 8 * i, t = lane & 3;
      if constexpr (D == 32) shared_words<8>(step + place(r, t >> 1) + (t & 1) * 8, k[i]);
      if constexpr (D == 64) shared_words<16>(step + place(r, t), k[i]);
      if constexpr (D == 128) {
        shared_words<16>(step + place(r, 2 * t), k[i]);
        shared_words<16>(step + place(r, 2 * t + 1), k[i] + 4);
      }
    }
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const uint32_t x0 = k[0][w] ^ 0x80808080u, x1 = k[1][w] ^ 0x80808080u;
      const uint32_t op[4] = {half_lo(x0), half_lo(x1), half_hi(x0), half_hi(x1)};
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int c = 0; c < QP; ++c) mma16816(z[n], op, q[n][c][w][0], q[n][c][w][1]);
    }
  }

  // scores to weights, in place; j: position of the step's first token; e: its block's scales
  __device__ __forceinline__ void weights(const AttnArgs &a, const float4 e, float (&z)[NQ][4], int j, int lane, int p_min,
                                          int p_max) {
    const bool whole = j + 15 <= p_min && (a.window <= 0 || j > p_max - a.window) && e.w != 0.f;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) z[n][i] = fmaf(z[n][i], rowf[n][i & 1] * e.x, e.y);
    if (!whole) {
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = j + (lane >> 2) + 8 * (i >> 1), pr = p[n][i & 1];
          const bool seen = at <= pr && (a.window <= 0 || at > pr - a.window) && e.w != 0.f;
          z[n][i] = seen ? z[n][i] : -INFINITY;
        }
    }
    bool rise = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) rise |= fmaxf(z[n][i], z[n][i + 2]) - m[n][i] > SLACK;
    if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = fmaxf(z[n][i], z[n][i + 2]);
#pragma unroll
          for (int d = 4; d <= 16; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const float to = fmaxf(m[n][i], reference(mx, HEAD, SLACK)), f = ex2(m[n][i] - to);
          m[n][i] = to;
          l[n][i] *= f;
#pragma unroll
          for (int c = 0; c < MT; ++c) {
            o[n][c][i] *= f;
            o[n][c][i + 2] *= f;
          }
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        z[n][i] = ex2(z[n][i] - m[n][i & 1]);
        l[n][i & 1] = fmaf(z[n][i], e.z, l[n][i & 1]);
      }
  }

  __device__ __forceinline__ void outputs(const float (&z)[NQ][4], uint32_t step, int lane) {
    uint32_t b[NQ][WP][2], v[4][VW];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      constexpr int VB = D / 8;  // bytes of a token's row that a lane needs
      const int r = 2 * (lane & 3) + (i & 1) + 8 * (i >> 1), at = (lane >> 2) * VB;
      shared_words<VB>(step + 16 * D + place(r, at >> 4) + (at & 15), v[i]);
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t hi = pack_half(z[n][2 * i], z[n][2 * i + 1]);
        b[n][0][i] = transpose8(hi);
        if constexpr (WP == 2) b[n][1][i] = transpose8(pack_rest(z[n][2 * i], z[n][2 * i + 1], hi));
      }
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      // four tokens' words -> for each element the pairs (token 2t, 2t + 1) and (2t + 8, 2t + 9)
      const uint32_t x0 = v[0][w] ^ 0x80808080u, x1 = v[1][w] ^ 0x80808080u;
      const uint32_t x2 = v[2][w] ^ 0x80808080u, x3 = v[3][w] ^ 0x80808080u;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t y0 = prmt(x0, x1, c ? 0x7362 : 0x5140), y1 = prmt(x2, x3, c ? 0x7362 : 0x5140);
        const uint32_t op[4] = {half_lo(y0), half_hi(y0), half_lo(y1), half_hi(y1)};
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          if constexpr (sizeof(T) == 4) {
            // tensor cores add with truncation, which drifts over many steps: the running sum is rounded to
            // nearest (58 sequences of 40700 tokens, error 4.0e-6 without; 16-bit calls: fold_sums)
            float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < WP; ++r) mma16816(y, op, b[n][r][0], b[n][r][1]);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[n][2 * w + c][r] += y[r];
          } else {
#pragma unroll
            for (int r = 0; r < WP; ++r) mma16816(o[n][2 * w + c], op, b[n][r][0], b[n][r][1]);
          }
        }
      }
    }
  }

  // O so far to a total in global memory (this thread's, THREADS floats from element to element, M last), and begun
  // anew; or, at a segment's end, back to registers
  __device__ __forceinline__ void fold(float *total, bool begun, bool last) {
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float *at = total + (size_t)((n * 2 + i) * (2 * MT + 1)) * THREADS;
        const float f = begun ? ex2(at[2 * MT * THREADS] - m[n][i]) : 0.f;
        at[2 * MT * THREADS] = m[n][i];
#pragma unroll
        for (int c = 0; c < 2 * MT; ++c) {
          float &x = o[n][c / 2][i + 2 * (c % 2)];
          const float y = begun ? fmaf(at[c * THREADS], f, x) : x;
          at[c * THREADS] = y;
          x = last ? y : 0.f;
        }
      }
  }

  // f grew by d: by RISE at most, or from 0 after blocks of zeros (O is 0), which then count with f - FAR as well
  __device__ __forceinline__ void raise(int d) {
    const float by = (float)max(0, d - FAR), f = ex2((float)d - by);
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (m[n][i] > LOWEST) m[n][i] += by;
        l[n][i] *= f;
      }
  }
};

// joins the sums of a cluster's CTAs (each the four warps' O in `so`, M and l in
// sm and sl) and writes the item's rows; the formula is join_kernel's
template <typename T, int D, int NQ>
__device__ __forceinline__ void join_cluster(const AttnArgs &a, const Seq &s, int tile, int kvh, float *so, float (*sm)[8 * NQ],
                                             float (*sl)[8 * NQ], const float *sf) {
  constexpr int R = 8 * NQ, PAD = D + 4;
  __shared__ float mine[3][R];  // M, f, l
  const int tid = threadIdx.x, size = gridDim.x, rank = blockIdx.x;
  for (int x = tid; x < R * (D / 4); x += THREADS) {  // the four warps' O into the first one's place
    float4 *y = reinterpret_cast<float4 *>(so + x / (D / 4) * PAD + x % (D / 4) * 4);
    constexpr int Q = R * PAD / 4;
    const float4 v0 = y[0], v1 = y[Q], v2 = y[2 * Q], v3 = y[3 * Q];
    y[0] = make_float4((v0.x + v1.x) + (v2.x + v3.x), (v0.y + v1.y) + (v2.y + v3.y), (v0.z + v1.z) + (v2.z + v3.z),
                       (v0.w + v1.w) + (v2.w + v3.w));
  }
  if (tid < R) {
    const float m = fmaxf(fmaxf(sm[0][tid], sm[1][tid]), fmaxf(sm[2][tid], sm[3][tid]));
    float l = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) l = fmaf(sl[i][tid], ex2(sm[i][tid] - m), l);
    mine[0][tid] = m;
    mine[1][tid] = sf[tid];
    mine[2][tid] = l;
  }
  cluster_sync();
  const int work = R * (D / 4), x0 = rank * work / size, x1 = (rank + 1) * work / size;
  for (int x = x0 + tid; x < x1; x += THREADS) {
    const int r = x / (D / 4), d = x % (D / 4) * 4, rho = tile * R + r;
    if (rho >= s.n * a.G) continue;
    // all CTAs' values at once: one remote latency (a rank past the size reads its own again, and is left out)
    float m[8], fc[8], lc[8], mg = LOWEST, ag = LOWEST, l = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
    uint4 v[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const uint32_t from = c < size ? c : rank;
      m[c] = ld_dsmem_f32(dsmem_addr(&mine[0][r], from));
      fc[c] = ld_dsmem_f32(dsmem_addr(&mine[1][r], from));
      lc[c] = ld_dsmem_f32(dsmem_addr(&mine[2][r], from));
      v[c] = ld_dsmem_v4(dsmem_addr(so + r * PAD + d, from));
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      mg = fmaxf(mg, m[c]);
      if (m[c] > LOWEST) ag = fmaxf(ag, m[c] - fc[c]);
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      if (c < size) {
        const float w = ex2(m[c] - mg);
        l = fmaf(lc[c], m[c] > LOWEST ? ex2((m[c] - ag) - fc[c]) : 1.f, l);  // (M - f alone rounds where scores pass 2^24)
        y[0] = fmaf(u2f(v[c].x), w, y[0]);
        y[1] = fmaf(u2f(v[c].y), w, y[1]);
        y[2] = fmaf(u2f(v[c].z), w, y[2]);
        y[3] = fmaf(u2f(v[c].w), w, y[3]);
      }
    }
    const float w = l == 0.f ? 0.f : 1.f / l, top = mg > LOWEST ? mg - ag : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = times_pow2(y[i] * w, top);
    store4<T>(static_cast<T *>(a.out) + ((size_t)(s.r0 + rho / a.G) * a.H + kvh * a.G + rho % a.G) * D + d, y);
  }
  cluster_sync();  // this CTA's sums are read until here
}

template <typename T, int D, int NQ>
__global__ void __launch_bounds__(THREADS, resident(DTYPE<T>, D, NQ)) attention_kernel(AttnArgs a) {
  constexpr int R = 8 * NQ, PAD = D + 4;
  __shared__ Meta meta;
  __shared__ long long scan[WARPS];
  __shared__ int found;
  __shared__ long long found_at;
  __shared__ Seq found_seq;
  __shared__ float sm[WARPS][R], sl[WARPS][R], sf[R];  // sf: f of each row
  extern __shared__ __align__(16) uint8_t ring[];  // [WARPS][STAGES] steps; then the warps' O [WARPS][R][PAD]
  after_previous_kernel();
  if (!a.split) next_kernel_may_start();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const long long cta = blockIdx.x;

  // where this CTA's share of the line of units begins: [lo, hi), in sequence b from unit `at` of b on
  int b, tile, kvh, u;
  long long lo = 0, hi = 0, total = 0, base = 0, grid = 1;
  Seq s;
  if (a.split) {
    const int per = (a.r.B + THREADS - 1) / THREADS, b0 = min(tid * per, a.r.B), b1 = min(b0 + per, a.r.B);
    long long mine = 0;
    for (int i = b0; i < b1; ++i) {
      const Seq x = seq_of<UNIT, 8 * NQ>(a, i);
      mine += (long long)x.units * x.tiles * a.c.KV;
    }
    long long upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const long long y = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += y;
    }
    if (lane == 31) scan[warp] = upto;
    __syncthreads();
    for (int i = 0; i < warp; ++i) upto += scan[i];
    for (int i = 0; i < WARPS; ++i) total += scan[i];
    grid = min((long long)gridDim.x, total);  // no CTA between two others is without a unit
    if (cta >= grid) return;
    lo = cta * total / grid;
    hi = (cta + 1) * total / grid;
    if (lo < upto && lo >= upto - mine) {
      long long x0 = upto - mine;
      int i = b0;
      Seq x = seq_of<UNIT, 8 * NQ>(a, i);
      while (i < b1 - 1 && lo >= x0 + (long long)x.units * x.tiles * a.c.KV) {
        x0 += (long long)x.units * x.tiles * a.c.KV;
        x = seq_of<UNIT, 8 * NQ>(a, ++i);
      }
      found = i;
      found_at = x0;
      found_seq = x;
    }
    __syncthreads();
    b = found;
    base = found_at;  // line index of sequence b's first unit
    s = found_seq;
    if (s.units == 0) return;  // only if lengths changed under the call
    const long long at = lo - base;
    u = (int)(at % s.units);
    const long long item = at / s.units;
    kvh = (int)(item % a.c.KV);
    tile = (int)(item / a.c.KV);
  } else {
    // grid: (cluster, KV head and tile, sequence); the cluster's size is a power of two
    const int shift = 31 - __clz(gridDim.x), rank = blockIdx.x;
    tile = blockIdx.y / a.c.KV;
    kvh = blockIdx.y - tile * a.c.KV;
    b = blockIdx.z;
    s = seq_of<UNIT, 8 * NQ>(a, b);
    if (tile >= s.tiles) return;  // the whole cluster
    u = (int)(((long long)rank * s.units) >> shift);
    lo = u;
    hi = ((long long)(rank + 1) * s.units) >> shift;
  }

  using W = Warp<T, D, NQ>;
  W w;
  const uint32_t mine = smem_u32(ring) + warp * (STAGES<D> * W::STEP);
  float *so = reinterpret_cast<float *>(ring);
  long long at = lo;
  do {
    // one segment: units [u, u1) of item (b, tile, kvh)
    const int u1 = (int)min((long long)s.units, u + (hi - at));
    const int first_rho = tile * R;
    int p_min = 0, p_max = 0;
    // the sequence's rows see positions see0 .. see1
    const int cap = a.r.width << a.c.lg_page, see0 = a.window > 0 ? max(0, max(s.p0, 0) - a.window + 1) : 0;
    const int see1 = min((long long)s.p0 + s.n - 1, (long long)cap - 1);
    const int chunk = ((META - 1) << a.c.lg_page) / UNIT;  // units whose pages are looked up together
    const long long head = (long long)kvh * a.c.page * D;
    // 16-bit calls: units after which O is added to its total, a whole number of chunks with FOLD / 2 tokens a warp
    const int spell = (FOLD / 2 / WTOK + chunk - 1) / chunk * chunk;
    auto place = [&]() { return a.total + (size_t)cta * (THREADS * NQ * (D / 4 + 2)) + tid; };
    int f = 0, f_first = 0;
    bool far = false;
    if (tid == 0) meta.f = 0;
    for (int c0 = u; c0 < u1; c0 += chunk) {
      const int c1 = min(u1, c0 + chunk);
      const int o0 = (s.u0 + c0) * UNIT >> a.c.lg_page, pages = (((s.u0 + c1) * UNIT - 1) >> a.c.lg_page) - o0 + 1;
      int id = -1;
      typename W::Query query;
      if (c0 > u) __syncthreads();  // every warp is done with the entries before
      if (sizeof(T) == 2 && a.total && c0 > u && (c0 - u) % spell == 0) w.fold(place(), c0 - u > spell, false);
      // on its way while the pages are looked up, where the registers allow it
      constexpr bool EARLY = NQ == 1 && D < 128;
      if (c0 == u && EARLY) w.load_query(query, a, s, tile, kvh, lane);
      if (tid < pages) {
        const int o = o0 + tid;
        if ((o + 1) << a.c.lg_page > see0 && o << a.c.lg_page <= see1) id = page_id(a.c, a.r, b, o);
        meta.off[tid] = max(id, 0) * a.c.page_stride + head;
      }
      __syncthreads();
      // fetches the warp's 16 tokens of unit c, if the chunk has it, into their ring step
      auto ring_step = [&](int c) { return mine + (c - c0) % STAGES<D> * W::STEP; };
      auto fetch = [&](int c) {
        if (c < c1) {
          const int j = (s.u0 + c) * UNIT + warp * WTOK;
          w.fetch(a, ring_step(c), meta.off[(j >> a.c.lg_page) - o0] + (j & (a.c.page - 1)) * D, lane);
        }
        copy_commit();
      };
#pragma unroll
      for (int i = 0; i < STAGES<D> - 1; ++i) fetch(c0 + i);
      int ek = 0, ev = 0;
      if (id >= 0) {
        ek = a.c.k_exp[id * a.c.exp_stride + kvh];
        ev = a.c.v_exp[id * a.c.exp_stride + kvh];
      }
      if (c0 == u) {
        if (!EARLY) w.load_query(query, a, s, tile, kvh, lane);
        w.start(query, a, s, tile, lane);
      }
      if (id >= 0 && ev != 255) atomicMax(&meta.f, ev);
      __syncthreads();
      const int f_old = f;
      f = meta.f;
      if (f_first == 0) f_first = f;
      if (tid < pages)
        meta.s[tid] = make_float4(pow2_e8m0(ek), ev == 255 ? __uint_as_float(0x7fc00000u) : (float)(ev - 127),
                                  ev == 255 ? 1.f : pow2_e8m0(min(127 + f - ev, 254)), id >= 0 ? 1.f : 0.f);
      far = f > f_first + RISE;
      if (__syncthreads_or(id >= 0 && ev < f - FAR) || (c0 > u && f_old == 0 && f > 0)) {
        // blocks of zeros are not far: these here count with f - FAR, the ones before, if f was 0, through raise
        for (int o = c0 > u && f_old == 0 ? (s.u0 + u) * UNIT >> a.c.lg_page : o0; o < o0 + pages && !far; ++o) {
          const int page = (o + 1) << a.c.lg_page > see0 && o << a.c.lg_page <= see1 ? page_id(a.c, a.r, b, o) : -1;
          const int e = page < 0 ? 255 : a.c.v_exp[page * a.c.exp_stride + kvh];
          if (e >= f - FAR) continue;
          far = __syncthreads_or(e > 0 || has_value(a, page, kvh, tid, THREADS));
          if (tid == 0 && o >= o0) {
            meta.s[o - o0].y = (float)(f - FAR - 127);
            meta.s[o - o0].z = pow2_e8m0(127 + FAR);
          }
        }
        __syncthreads();
      }
      if (far) {  // (copies on their way land before the ring's memory is used otherwise)
        copy_wait<0>();
        break;
      }
      if (c0 > u && f > f_old) w.raise(f - f_old);
      if (c0 == u) {
        p_min = p_max = w.p[0][0];  // of the tile's rows
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            p_min = min(p_min, w.p[n][i]);
            p_max = max(p_max, w.p[n][i]);
          }
        p_min = __reduce_min_sync(0xffffffffu, p_min);
        p_max = __reduce_max_sync(0xffffffffu, p_max);
      }
      for (int c = c0; c < c1; ++c) {
        float z[NQ][4];
        const int j = (s.u0 + c) * UNIT + warp * WTOK;
        const float4 e = meta.s[(j >> a.c.lg_page) - o0];
        const uint32_t step = ring_step(c);
        copy_wait<STAGES<D> - 2>();
        __syncwarp();  // every lane's copies of this step are there, and its reads of the last one done
        w.scores(z, step, lane);
        fetch(c + STAGES<D> - 1);  // into the step that the last iteration read
        w.weights(a, e, z, j, lane, p_min, p_max);
        w.outputs(z, step, lane);
      }
      copy_wait<0>();
    }
    if (sizeof(T) == 2 && a.total && !far && u1 - u > spell) w.fold(place(), true, true);
    if (u == u1) {  // no units: nothing to add, or an item of zeros
      typename W::Query none = {};
      w.start(none, a, s, tile, lane);
    }
    if (far) {  // the segment anew, a row a warp; the other warps' places hold nothing
      __syncthreads();
      const int j0 = (s.u0 + u) * UNIT, j1 = (s.u0 + u1) * UNIT, lift = far_lift(a, b, kvh, j0, j1, lane);
      for (int r = warp; r < R && first_rho + r < s.n * a.G; r += WARPS) {
        const int rho = first_rho + r;
        float m, l, o[D / 32];
        far_row<T, D>(a, b, kvh, static_cast<const T *>(a.q) + (s.r0 + rho / a.G) * a.ld + (size_t)(kvh * a.G + rho % a.G) * D,
                      row_pos(a, s, rho), j0, j1, lift, lane, m, l, o);
        // O to about 2^20 and M as much higher, which is where the other records' M stand (zeros: far below)
        float top = 0.f;
#pragma unroll
        for (int d = 0; d < D / 32; ++d) top = fmaxf(top, fabsf(o[d]));
        top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
        const float at = m + (top > 0.f ? floorf(log2f(top)) - 20.f : -300.f), shift = m > LOWEST ? at - m : 0.f;  // (as it rounds)
#pragma unroll
        for (int i = 0; i < WARPS; ++i) {
#pragma unroll
          for (int d = 0; d < D / 32; ++d) so[(i * R + r) * PAD + lane * (D / 32) + d] = i ? 0.f : times_pow2(o[d], -shift);
          sm[i][r] = i || m == LOWEST ? LOWEST : at;
          sl[i][r] = i ? 0.f : l;
        }
        sf[r] = shift + (float)lift;
      }
    } else {
      // the warps' sums, brought to a common M
      if (tid < R) sf[tid] = (float)(f - 127);
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int d = 4; d <= 16; d *= 2) w.l[n][i] += __shfl_xor_sync(0xffffffffu, w.l[n][i], d);
          if (g == 0) {
            sm[warp][8 * n + 2 * t + i] = w.m[n][i];
            sl[warp][8 * n + 2 * t + i] = w.l[n][i];
          }
        }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = 8 * n + 2 * t + i;
          const float f = ex2(w.m[n][i] - fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r])));
#pragma unroll
          for (int c = 0; c < W::MT; ++c)
            *reinterpret_cast<float2 *>(so + (warp * R + r) * PAD + g * (D / 8) + 2 * c) =
                make_float2(w.o[n][c][i] * f, w.o[n][c][i + 2] * f);
        }
    }
    __syncthreads();
    if (!a.split && gridDim.x > 1) {
      join_cluster<T, D, NQ>(a, s, tile, kvh, so, sm, sl, sf);
      return;
    }
    const bool whole = u == 0 && u1 == s.units;
    float *rec = whole ? nullptr : a.part + (cta * 2 + (u == 0 ? 1 : 0)) * (size_t)(R * (D + 3));
    for (int x = tid; x < R * (D / 4); x += THREADS) {
      const int r = x / (D / 4), d = x % (D / 4) * 4, rho = first_rho + r;
      if (rho >= s.n * a.G) continue;
      const float mx = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
      float l = 0.f;
#pragma unroll
      for (int i = 0; i < WARPS; ++i) l = fmaf(sl[i][r], ex2(sm[i][r] - mx), l);
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        y[i] = (so[r * PAD + d + i] + so[(R + r) * PAD + d + i]) + (so[(2 * R + r) * PAD + d + i] + so[(3 * R + r) * PAD + d + i]);
      if (whole) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = l == 0.f ? 0.f : times_pow2(y[i] / l, sf[r]);
        store4<T>(static_cast<T *>(a.out) + ((size_t)(s.r0 + rho / a.G) * a.H + kvh * a.G + rho % a.G) * D + d, y);
      } else {
        *reinterpret_cast<float4 *>(rec + r * D + d) = make_float4(y[0], y[1], y[2], y[3]);
        if (d == 0) {
          rec[R * D + r] = mx;
          rec[R * (D + 1) + r] = l;
          rec[R * (D + 2) + r] = sf[r];
        }
      }
    }
    if (!whole && u == 0 && tid == 0) {
      // the item ends at line index base + its units; the CTA that holds its last one
      const long long end = at + s.units;
      a.desc[((size_t)b * a.tiles + tile) * a.c.KV + kvh] = make_int2((int)cta, (int)((end * grid - 1) / total));
    } else if (a.split && whole && tid == 0) {
      a.desc[((size_t)b * a.tiles + tile) * a.c.KV + kvh] = make_int2((int)cta, (int)cta);
    }
    at += u1 - u;
    if (at >= hi) break;
    u = 0;
    if (++kvh == a.c.KV) {
      kvh = 0;
      if (++tile == s.tiles) {
        tile = 0;
        do {
          if (++b == a.r.B) return;  // (lengths changed under the call)
          s = seq_of<UNIT, 8 * NQ>(a, b);
        } while (s.units == 0);
      }
    }
    __syncthreads();  // so, sm and sl are read until here
  } while (true);
}

// joins the records of a row that several CTAs share, in their order: with
// Mg = max M and Ag = max (M - f) over the records,
//   out = 2^(Mg - Ag) sum O 2^(M - Mg) / sum l 2^(M - f - Ag).
// One CTA a row: its threads are D / 4 columns by THREADS / (D / 4) record
// slices. Writes the zeros of sequences without visible tokens.
template <typename T, int D, int NQ>
__global__ void __launch_bounds__(THREADS) join_kernel(AttnArgs a) {
  constexpr int R = 8 * NQ, C = D / 4, SLICES = THREADS / C;
  __shared__ float red[2][WARPS], wo[THREADS];
  __shared__ float4 part[SLICES][C];
  __shared__ float den[WARPS];
  after_previous_kernel();
  const int r = blockIdx.x % R, kvh = blockIdx.x / R % a.c.KV, tile = blockIdx.x / R / a.c.KV, b = blockIdx.y;
  const int tid = threadIdx.x, col = tid % C, slice = tid / C, rho = tile * R + r;
  const Seq s = seq_of<UNIT, 8 * NQ>(a, b);
  if (rho >= s.n * a.G) return;
  T *dst = static_cast<T *>(a.out) + ((size_t)(s.r0 + rho / a.G) * a.H + kvh * a.G + rho % a.G) * D + 4 * col;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  if (s.units == 0) {
    if (slice == 0) store4<T>(dst, reinterpret_cast<const float(&)[4]>(y));
    return;
  }
  const int2 span = a.desc[((size_t)b * a.tiles + tile) * a.c.KV + kvh];
  if (span.x == span.y) return;
  auto record = [&](int c) { return a.part + ((size_t)c * 2 + (c == span.x ? 1 : 0)) * (size_t)(R * (D + 3)); };
  float mg = LOWEST, ag = LOWEST, l = 0.f;
  for (int c = span.x + tid; c <= span.y; c += THREADS) {
    const float *q = record(c) + R * D + r;
    mg = fmaxf(mg, q[0]);
    if (q[0] > LOWEST) ag = fmaxf(ag, q[0] - q[2 * R]);
  }
#pragma unroll
  for (int d = 16; d >= 1; d /= 2) {
    mg = fmaxf(mg, __shfl_xor_sync(0xffffffffu, mg, d));
    ag = fmaxf(ag, __shfl_xor_sync(0xffffffffu, ag, d));
  }
  if ((tid & 31) == 0) {
    red[0][tid >> 5] = mg;
    red[1][tid >> 5] = ag;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    mg = fmaxf(mg, red[0][i]);
    ag = fmaxf(ag, red[1][i]);
  }
  for (int c0 = span.x; c0 <= span.y; c0 += THREADS) {
    const int n = min(THREADS, span.y - c0 + 1);
    if (tid < n) {
      const float *q = record(c0 + tid) + R * D + r;
      wo[tid] = ex2(q[0] - mg);
      l = fmaf(q[R], q[0] > LOWEST ? ex2((q[0] - ag) - q[2 * R]) : 1.f, l);
    }
    __syncthreads();
#pragma unroll 4
    for (int c = slice; c < n; c += SLICES) {
      const float4 v = *reinterpret_cast<const float4 *>(record(c0 + c) + r * D + 4 * col);
      const float f = wo[c];
      y.x = fmaf(v.x, f, y.x);
      y.y = fmaf(v.y, f, y.y);
      y.z = fmaf(v.z, f, y.z);
      y.w = fmaf(v.w, f, y.w);
    }
    __syncthreads();
  }
  part[slice][col] = y;
#pragma unroll
  for (int d = 16; d >= 1; d /= 2) l += __shfl_xor_sync(0xffffffffu, l, d);
  if ((tid & 31) == 0) den[tid >> 5] = l;
  __syncthreads();
  if (slice) return;
  for (int i = 1; i < SLICES; ++i) {
    const float4 v = part[i][col];
    y = make_float4(y.x + v.x, y.y + v.y, y.z + v.z, y.w + v.w);
  }
  l = den[0] + den[1] + den[2] + den[3];
  const float f = l == 0.f ? 0.f : 1.f / l, top = mg > LOWEST ? mg - ag : 0.f;
  const float out[4] = {times_pow2(y.x * f, top), times_pow2(y.y * f, top), times_pow2(y.z * f, top), times_pow2(y.w * f, top)};
  store4<T>(dst, out);
}

struct Plan {
  int prompt, nq, tiles, split, cluster, grid;
  size_t desc, total, bytes;  // total: where the workspace's `total` begins, 0 without
};

// rows of a tile: 8 or 16; 24 where that saves a tile and the registers suffice
int row_tiles(long long rows, int dtype, int D, int &nq) {
  nq = rows <= 8 ? 1 : 2;
  if (nq == 2 && !(dtype == LBC_F32 && D == 128) && (rows + 23) / 24 < (rows + 15) / 16) nq = 3;
  return (int)((rows + 8 * nq - 1) / (8 * nq));
}

// Which kernel, and how its work is cut.
//   prompt      Measured in bf16 at D = 128: the prompt kernel takes 1.35 us a
//               wave of its CTAs and 64 tokens, this one 1.3 us for 2 SMs' worth of
//               units; so it takes over when its waves are the fewer. Other types
//               and sizes go by the same rule, unmeasured; it leaves out that a tile
//               here goes through all that its sequence sees, the causal or windowed
//               part of its own rows or not.
//   cluster     a CTA goes through at most 16 units (1024 tokens), and a wave
//               holds the clusters of every item where there is more than one CTA
//   split       otherwise; more CTAs than SMs only where each gets THIN units of
//               the longest possible sequences: below, a CTA's start and the
//               records that it adds to the join cost more than it saves.
//               Measured with 1 / 3 / 5 / 7: one sequence of 30000 tokens, 2 KV
//               heads 19.8 / 15.6 / 15.1 / 13.5 us; two of up to 16000, 8 KV
//               heads 21.1 / 21.2 / 21.2 / 23.0
constexpr int THIN = 6;
Plan plan_of(const Pool &c, int dtype, int width, int B, int N, int most, int H, int window, int sms) {
  Plan p{};
  const long long rows = (long long)std::max(most, 1) * (H / c.KV);  // (max_tokens 0: one CTA a sequence records the rows left out)
  p.tiles = row_tiles(rows, dtype, c.D, p.nq);
  const long long items = (long long)B * c.KV * p.tiles;
  const int high = prompt_rows(dtype, c.D);
  const long long waves = ((long long)B * c.KV * ((rows + high - 1) / high) + sms - 1) / sms;
  p.prompt = rows > 24 && waves * 2 * sms <= items;
  long long len = (long long)width << c.lg_page;
  if (window > 0) len = std::min(len, (long long)window + most + UNIT);
  if (p.prompt) {
    p.bytes = fold_sums(dtype, len) ? (size_t)N * H * total_row(c.D) * sizeof(float) : 0;
    return p;
  }
  const long long units = (len + UNIT - 1) / UNIT;
  const long long wave = (long long)resident(dtype, c.D, p.nq) * sms;
  p.cluster = 1;
  while (p.cluster < 8 && 2 * p.cluster <= units && 2 * p.cluster * items <= wave) p.cluster *= 2;
  p.split = units > 16 * p.cluster;
  p.grid = (int)std::min<long long>(p.split ? std::min(wave, std::max<long long>(items * units / THIN, sms)) : items * p.cluster, 0x7fffffff);
  p.desc = p.split ? ((size_t)items * sizeof(int2) + 255) / 256 * 256 : 0;
  p.bytes = p.split ? p.desc + (size_t)p.grid * 2 * 8 * p.nq * (c.D + 3) * sizeof(float) : 0;
  if (p.split && fold_sums(dtype, len / 2)) {
    p.total = (p.bytes + 255) / 256 * 256;
    p.bytes = p.total + (size_t)p.grid * THREADS * p.nq * (c.D / 4 + 2) * sizeof(float);
  }
  return p;
}

template <typename T, int D, int NQ>
void launch(const AttnArgs &a, const Plan &p, cudaStream_t st) {
  constexpr int smem = std::max(WARPS * STAGES<D> * Warp<T, D, NQ>::STEP, (int)sizeof(float) * WARPS * 8 * NQ * (D + 4));
  static std::atomic<uint64_t> allowed{0};
  allow_smem(attention_kernel<T, D, NQ>, smem, allowed);
  launch_chained(attention_kernel<T, D, NQ>, p.split ? dim3(p.grid) : dim3(p.cluster, a.c.KV * p.tiles, a.r.B), THREADS, smem,
                 p.split ? 1 : p.cluster, st, a);
  if (p.split) launch_chained(join_kernel<T, D, NQ>, dim3(8 * NQ * a.c.KV * a.tiles, a.r.B), THREADS, 0, 1, st, a);
}
template <typename T, int D>
void launch(const AttnArgs &a, const Plan &p, cudaStream_t st) {
  if (p.nq == 1) launch<T, D, 1>(a, p, st);
  else if (p.nq == 2) launch<T, D, 2>(a, p, st);
  else if constexpr (!(sizeof(T) == 4 && D == 128)) launch<T, D, 3>(a, p, st);
}
template <typename T>
void launch(const AttnArgs &a, const Plan &p, cudaStream_t st) {
  if (a.c.D == 32) launch<T, 32>(a, p, st);
  else if (a.c.D == 64) launch<T, 64>(a, p, st);
  else launch<T, 128>(a, p, st);
}

}  // namespace
}  // namespace kv8
}  // namespace lbc

using namespace lbc;
using namespace lbc::kv8;

extern "C" {

size_t lbc_kv8_attention_workspace(const lbc_kv8 *c, int dtype, int table_width, int B, int N, int max_tokens, int H,
                                   int window) {
  Pool p;
  int *status = nullptr, sms = 0;
  if (check_pool(c, p) || device_ready(&status, &sms) || table_width <= 0 || B <= 0 || H <= 0 || H % p.KV || max_tokens < 0 || N < 0)
    return 0;
  return plan_of(p, dtype, table_width, B, N, max_tokens, H, window, sms).bytes;
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
  if (H <= 0 || H % a.c.KV || H > 65535 || (long long)max_tokens * H > 0x7fffffff)
    return refuse("kv8_attention: H must be a multiple of the KV heads");
  if ((long long)max_tokens * (H / a.c.KV) > 128LL * 65535) return refuse("kv8_attention: too many rows a sequence");
  if (N == 0) return 0;
  if (!q || !out) return refuse("kv8_attention: NULL argument");
  if (ld < (long long)H * a.c.D || ld * (dtype == LBC_F32 ? 4 : 2) % 16) return refuse("kv8_attention: bad row stride");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15)
    return refuse("kv8_attention: q and out must be 16-byte aligned");
  a.q = q; a.ld = ld; a.out = out; a.H = H; a.G = H / a.c.KV; a.window = window;
  a.scale_log2 = scale * 1.4426950408889634f;
  const Plan p = plan_of(a.c, dtype, table_width, B, N, max_tokens, H, window, sms);
  if (p.bytes && (!workspace || workspace_bytes < p.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255)))
    return refuse("kv8_attention: workspace too small or not 256-byte aligned");
  a.tiles = p.tiles;
  a.split = p.split;
  a.desc = static_cast<int2 *>(workspace);
  a.total = p.prompt && p.bytes ? static_cast<float *>(workspace)
            : p.total           ? reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + p.total)
                                : nullptr;
  a.part = p.split ? reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + p.desc) : nullptr;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.prompt) launch_prompt(a, dtype, st);
  else if (dtype == LBC_F32) launch<float>(a, p, st);
  else if (dtype == LBC_BF16) launch<__nv_bfloat16>(a, p, st);
  else launch<__half>(a, p, st);
  return launched("kv8_attention");
}

}  // extern "C"
