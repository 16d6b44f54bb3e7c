// Causal grouped-query attention over the paged 8-bit KV cache for many rows
// (prompts and prompt chunks), on tcgen05.
//
// A CTA takes 256 rows (token t, head g of the group: row t G + g) of one
// sequence and KV head as two tiles of 128 (fp32 at D = 128: one), and runs through the visible tokens
// 64 at a time:
//   warps 0-7   a thread a row: scores from tensor memory, scale, mask, running
//               reference M, weights 2^(t - M), sums l; O is rescaled only when a
//               row's maximum has risen by more than 2^3 (fp32: added to a total)
//   warps 8-11  codes to fp16 operand tiles (exact; keys K-major as they lie, values
//               transposed 8 x 8 in registers), one conversion for both row tiles
//   warp 12     S = Q K^T, both operands in shared memory, S in two buffers so that
//               the scores of a step are ready when the weights of the last are done
//   warp 13     O += P V, P (fp16) in tensor memory where S was
//   warp 14     codes from global memory into a ring, up to 4 steps ahead (bulk copies)
//   warp 15     block scales, 8 steps at a time
// Scales, M, l and f are those of the few-row kernel (kv8_attention.cu); queries
// are scaled into fp16's range per row, fp32 ones in two pieces, and weights of
// fp32 and fp16 calls in two pieces (twice the products).
//
// Bound: the row warps' own chain of a step (tensor-memory load, scale, maximum,
// vote, exponentials, store): 2500-2600 cycles, of which the tensor pipe works
// 1288 and the exponential unit 1024. Two prompts to 4096 tokens, 32 heads, 8 KV
// heads of 128, bf16: 213-218 us, 680-690 TFLOP/s; 2048 fp32 tokens after 2047, 14
// heads of 64: 106 us. 64 tokens a step and not 128, so that two steps' scores fit
// tensor memory beside two row tiles' outputs (128 with one: 293 us); two row
// tiles share each conversion of the codes.
#include <algorithm>
#include <cstdio>

#include "kernels.h"
#include "kv8_attn.cuh"
#include "tc.cuh"

namespace lbc {
namespace kv8 {
namespace {

constexpr int NT = 64;        // tokens a step
constexpr int TILE = 128;     // rows of a row tile
constexpr int W_DEQ = 8, W_MMA = 12, W_COPY = 14, W_SCALE = 15, THREADS = 16 * 32;
// registers a thread of the three kinds of warpgroups, out of 128 at launch
constexpr int R_ROWS = 184, R_DEQ = 72, R_REST = 64;
static_assert(256 * R_ROWS + 128 * (R_DEQ + R_REST) <= THREADS * 128, "a block's registers");
constexpr int META = 8;       // steps whose block scales are looked up together; two such sets are kept
constexpr int RAW = 4;        // steps whose codes are in flight or waiting
// added to a set's f from where the value exponents lie farther apart than the row warps' sums allow (kv8_attn.cuh: FAR)
constexpr int APART = 1024;
// weights: M is the maximum (rounded up) less 12, left alone up to 2^15
constexpr float HEAD = 12.f, SLACK = 15.f;

struct Scales {
  float4 g[META][NT / 16];  // of each 16 tokens: 2^(ek - 127), b = ev - 127, 2^(f - b), 1 if the page exists
  int f, all, pad[2];       // f: largest value exponent so far; all: every page of the set exists
};

// Full / empty pairs of the rings (two stages each; phase j >> 1), S and P full
// by row tile and buffer, outputs done by row tile and step parity. A parity
// wait only tells neighbouring phases apart: every wait below follows from an
// earlier one that its barrier is at most one phase behind.
struct Shared {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], raw_full[RAW], raw_empty[RAW], s_full[2][2], p_full[2][2], pv_done[2][2], meta_full[2], meta_empty[2], q_full, s_fin, fin;
  uint32_t tmem;
  int abort;  // a wait ran out
  Scales meta[2];
};

// operand tiles, in bytes. K-major without swizzle: 8 rows x 16 bytes are one
// core matrix; LBO steps along K, SBO along the rows. The strides carry a
// pad that spreads a warp's stores over the banks.
template <typename T, int D>
struct Lay {
  // row tiles of a CTA. Tensor cores add with truncation, which over thousands of
  // tokens shows in fp32 outputs: fp32 calls begin O anew in each step and add it
  // to a total (rounded to nearest, also in tensor memory; adding every fourth
  // step only drifts by 1.1e-6 and is no faster, 109 to 106 us); at D = 128 the
  // total leaves room for one row tile. 16-bit outputs need it seldom, in the
  // workspace (kv8_attn.cuh: fold_sums).
  static constexpr bool FOLD = sizeof(T) == 4;
  static constexpr int RT = FOLD && D == 128 ? 1 : 2, ROWS = RT * TILE;
  static constexpr int QP = QUERY_PIECES<T>, WP = WEIGHT_PIECES<T>;
  static constexpr int Q_LBO = TILE / 8 * 128 + 16, Q_BYTES = D / 8 * Q_LBO;
  static constexpr int K_LBO = NT / 8 * 128 + 16 * (128 / D), K_BYTES = D / 8 * K_LBO;
  static constexpr int V_SBO = 144, V_LBO = D / 8 * V_SBO, V_BYTES = NT / 8 * V_LBO;
  static constexpr int K_OFF = RT * QP * Q_BYTES, V_OFF = K_OFF + 2 * K_BYTES, R_BYTES = 2 * NT * D,
                       R_OFF = (V_OFF + 2 * V_BYTES + 127) / 128 * 128, S_OFF = R_OFF + RAW * R_BYTES;
  static constexpr int SMEM = S_OFF + (int)sizeof(Shared);
  // position along K of the 8 elements from 16 c + 8 h on (the order is free, and the same in Q and K)
  __device__ static int chunk(int c, int h) { return h * (D / 16) + c; }
};

template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// adds a row's O (16 elements from c on: get, by the whole warp) to its total, D floats and the M that they stand at,
// brought to M = m
template <int D, typename Get>
__device__ __forceinline__ void add_total(float *total, bool there, bool begun, float m, const Get &get) {
  float f = 0.f;
  if (there) {
    if (begun) f = ex2(total[D] - m);
    total[D] = m;
  }
#pragma unroll
  for (int c = 0; c < D; c += 16) {
    uint32_t o[16];
    get(c, o);
    if (!there) continue;
#pragma unroll
    for (int k = 0; k < 16; k += 4) {
      float4 *t = reinterpret_cast<float4 *>(total + c + k);
      float4 y = make_float4(u2f(o[k]), u2f(o[k + 1]), u2f(o[k + 2]), u2f(o[k + 3]));
      if (begun) {
        const float4 x = *t;
        y = make_float4(fmaf(x.x, f, y.x), fmaf(x.y, f, y.y), fmaf(x.z, f, y.z), fmaf(x.w, f, y.w));
      }
      *t = y;
    }
  }
}

// TOTAL: a 16-bit call that can see so many tokens that O is kept in a total (kv8_attn.cuh: fold_sums); an instance of its
// own, because the test for it in the other's loop costs 1 to 7 % (prompts to 4096 tokens: 215 us, 217 to 231 with it)
template <typename T, int D, bool TOTAL>
__global__ void __launch_bounds__(THREADS, 1) prompt_kernel(AttnArgs a) {
  using L = Lay<T, D>;
  extern __shared__ __align__(128) uint8_t smem[];
  Shared &sh = *reinterpret_cast<Shared *>(smem + L::S_OFF);
  after_previous_kernel();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.x, b = blockIdx.y, tile = gridDim.z - 1 - blockIdx.z;  // late rows, the longest, first
  const Seq s = seq_of<NT, L::ROWS>(a, b);
  if (tile >= s.tiles) return;
  const int rho0 = tile * L::ROWS, rho1 = min(rho0 + L::ROWS, s.n * a.G) - 1;
  const long long cap = (long long)a.r.width << a.c.lg_page;
  const long long p_first = max((long long)s.p0 + rho0 / a.G, 0LL), p_last = min((long long)s.p0 + rho1 / a.G, cap - 1);
  const long long see0 = a.window > 0 ? max(0LL, p_first - a.window + 1) : 0;
  const int t0 = (int)(see0 / NT), steps = p_last >= see0 ? (int)(p_last / NT) - t0 + 1 : 0;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.k_full[i], 128);
      mbar_init(&sh.v_full[i], 128);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_empty[i], 1);
      mbar_init(&sh.meta_full[i], 1);
      mbar_init(&sh.meta_empty[i], 4 * L::RT);
      for (int j = 0; j < 2; ++j) {
        mbar_init(&sh.pv_done[i][j], 1);
        mbar_init(&sh.s_full[i][j], 1);
        mbar_init(&sh.p_full[i][j], TILE);
      }
    }
    for (int i = 0; i < RAW; ++i) {
      mbar_init(&sh.raw_full[i], 1);
      mbar_init(&sh.raw_empty[i], 4);
    }
    mbar_init(&sh.q_full, L::ROWS);
    mbar_init(&sh.s_fin, 1);
    mbar_init(&sh.fin, 1);
    sh.abort = 0;
    fence_mbar_init();
  }
  if (warp == W_MMA) {
    tc::alloc(&sh.tmem, 512);
    tc::relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = sh.tmem, base = smem_u32(smem);
  volatile int *abort = &sh.abort;
  // a wait of a whole warp: every lane goes on, or (time limit, recorded) none;
  // a wait that ran out anywhere ends the ones that are not yet over
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (__all_sync(0xffffffffu, mbar_poll(bar, parity))) return true;
    const bool ok = !*abort && mbar_wait_polling(bar, parity, a.r.status);
    if (__all_sync(0xffffffffu, ok)) return true;
    *abort = 1;
    return false;
  };
  constexpr int anew = TOTAL ? kv8::FOLD / NT - 1 : 0x7fffffff;  // O begins anew at steps j with j & anew == 0
  // tensor memory: S (and P in its place) of row tile i, buffer j; O of row tile i; its total
  auto s_col = [&](int i, int j) { return tmem + (2 * i + j) * NT; };
  auto o_col = [&](int i) { return tmem + 2 * L::RT * NT + i * D; };
  auto t_col = [&](int i) { return tmem + 2 * L::RT * NT + (L::RT + i) * D; };

  if (warp == W_MMA) {
    // ------------------------------------------------------------ scores
    reg_dec<R_REST>();
    if (lane == 0 && steps > 0 && mbar_wait_polling(&sh.q_full, 0, a.r.status)) {
      const uint64_t qd = tc::smem_desc(base, L::Q_LBO, 128);
      for (int j = 0; j < steps && !*abort; ++j) {
        const int st = j & 1;
        bool ok = mbar_wait_polling(&sh.k_full[st], (j >> 1) & 1, a.r.status);
        const uint64_t kd = tc::smem_desc(base + L::K_OFF + st * L::K_BYTES, L::K_LBO, 128);
#pragma unroll
        for (int i = 0; i < L::RT; ++i) {
          // S goes where the weights of step j - 2 were
          if (j > 1) ok = ok && mbar_wait_polling(&sh.pv_done[i][st], ((j >> 1) & 1) ^ 1u, a.r.status);
          if (!ok) break;
          tc::fence_after_sync();
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int c = 0; c < L::QP; ++c)
              tc::mma_f16_ss(s_col(i, st), qd + (uint64_t)((i * L::QP + c) * L::Q_BYTES + 2 * k * L::Q_LBO) / 16,
                             kd + (uint64_t)(2 * k * L::K_LBO) / 16, tc::idesc_f16_f32(NT), k + c > 0);
          tc::commit(&sh.s_full[i][st]);
        }
        if (!ok) {
          *abort = 1;
          break;
        }
        tc::commit(&sh.k_empty[st]);
      }
      tc::commit(&sh.s_fin);
      mbar_wait_polling(&sh.s_fin, 0, a.r.status);
    }
  } else if (warp == W_MMA + 1) {
    // ------------------------------------------------------------ outputs
    reg_dec<R_REST>();
    if (lane == 0 && steps > 0) {
      for (int j = 0; j < steps && !*abort; ++j) {
        const int st = j & 1;
        const uint32_t ph = (j >> 1) & 1;
        bool ok = mbar_wait_polling(&sh.v_full[st], ph, a.r.status);
        const uint64_t vd = tc::smem_desc(base + L::V_OFF + st * L::V_BYTES, L::V_LBO, L::V_SBO);
#pragma unroll
        for (int i = 0; i < L::RT; ++i) {
          ok = ok && mbar_wait_polling(&sh.p_full[i][st], ph, a.r.status);
          if (!ok) break;
          tc::fence_after_sync();
#pragma unroll
          for (int c = L::WP - 1; c >= 0; --c)  // small pieces first: the sum they are cut to is small
#pragma unroll
            for (int k = 0; k < NT / 16; ++k)
              tc::mma_f16_ts(o_col(i), s_col(i, st) + 8 * k + NT / 2 * c, vd + (uint64_t)(2 * k * L::V_LBO) / 16,
                              tc::idesc_f16_f32(D), k > 0 || c < L::WP - 1 || (!L::FOLD && (j & anew) != 0));
          tc::commit(&sh.pv_done[i][st]);
        }
        if (!ok) {
          *abort = 1;
          break;
        }
        tc::commit(&sh.v_empty[st]);
      }
      tc::commit(&sh.fin);
      mbar_wait_polling(&sh.fin, 0, a.r.status);
    }
  } else if (warp == W_COPY) {
    // ------------------------------------------------------------ codes to the raw ring
    reg_dec<R_REST>();
    if (lane == 0 && steps > 0) {
      const int o_lo = (int)(see0 >> a.c.lg_page), o_hi = (int)(p_last >> a.c.lg_page);  // pages that the rows see
      const int32_t *ids = a.r.table + (size_t)b * a.r.width;
      const long long head = (long long)kvh * a.c.page * D;
      const int run = min(a.c.page, NT);  // tokens that lie together
      const uint64_t keep = policy_evict_normal();
      int j = 0;
      for (; j < steps && !*abort; ++j) {
        const int rs = j % RAW;
        if (!mbar_wait_polling(&sh.raw_empty[rs], (j / RAW & 1) ^ 1u, a.r.status)) {
          *abort = 1;
          break;
        }
        uint8_t *dst = smem + L::R_OFF + rs * L::R_BYTES;
        mbar_expect_tx(&sh.raw_full[rs], L::R_BYTES);
        for (int k = 0; k < NT; k += run) {
          // positions that no row sees take a neighbouring page's codes (they are masked), bad ids page 0's
          const int pos = (t0 + j) * NT + k, id = ids[min(max(pos >> a.c.lg_page, o_lo), o_hi)];
          const long long off = ((unsigned)id < (unsigned)a.c.pages ? id : 0) * a.c.page_stride + head + (pos & (a.c.page - 1)) * D;
          bulk_g2s(dst + k * D, a.c.k + off, run * D, &sh.raw_full[rs], keep);
          bulk_g2s(dst + (NT + k) * D, a.c.v + off, run * D, &sh.raw_full[rs], keep);
        }
      }
      // copies in flight land before the block's shared memory goes
      for (int k = max(0, j - RAW); k < j; ++k)
        if (!mbar_wait_polling(&sh.raw_full[k % RAW], (k / RAW) & 1, a.r.status)) break;
    }
  } else if (warp == W_SCALE) {
    // ------------------------------------------------------------ block scales, a lane 16 tokens of META steps
    reg_dec<R_REST>();
    const int o_lo = (int)(see0 >> a.c.lg_page), o_hi = (int)(p_last >> a.c.lg_page);
    const int32_t *ids = a.r.table + (size_t)b * a.r.width;
    int f = 0, f_first = 0, far = 0;  // largest value exponent so far (255 left out), and of the first set
    for (int j = 0; j < steps; j += META) {
      const int set = j / META & 1;
      const int id = ids[min(max(((t0 + j) * NT + lane * 16) >> a.c.lg_page, o_lo), o_hi)];
      const bool there = (unsigned)id < (unsigned)a.c.pages;
      if (!there) set_status(a.r.status, LBC_ERR_PAGE);
      const int ek = there ? a.c.k_exp[id * a.c.exp_stride + kvh] : 0, ev = there ? a.c.v_exp[id * a.c.exp_stride + kvh] : 0;
      const int f_old = f;
      f = max(f, __reduce_max_sync(0xffffffffu, ev == 255 ? 0 : ev));
      if (f_first == 0) f_first = f;
      if (f > f_first + RISE) far = APART;
      const int all = __all_sync(0xffffffffu, there);
      int at = ev;
      if (__any_sync(0xffffffffu, there && ev < f - FAR) || (j > 0 && f_old == 0 && f > 0)) {
        // blocks of zeros are not far: these here count with f - FAR, the ones before, if f was 0, by way of M
        const int o0 = (t0 + j) * NT >> a.c.lg_page, o1 = min(((t0 + j + META) * NT - 1) >> a.c.lg_page, o_hi);
        for (int o = j > 0 && f_old == 0 ? o_lo : max(o0, o_lo); o <= o1 && !far; ++o) {
          const int page = ids[o];
          const int e = (unsigned)page >= (unsigned)a.c.pages ? 255 : a.c.v_exp[page * a.c.exp_stride + kvh];
          if (e < f - FAR && __any_sync(0xffffffffu, e > 0 || has_value(a, page, kvh, lane, 32))) far = APART;
        }
        at = max(ev, f - FAR);
      }
      if (!wait(&sh.meta_empty[set], (j / META >> 1 & 1) ^ 1u)) break;
      sh.meta[set].g[lane / (NT / 16)][lane % (NT / 16)] =
          make_float4(pow2_e8m0(ek), ev == 255 ? __uint_as_float(0x7fc00000u) : (float)(at - 127),
                      ev == 255 ? 1.f : pow2_e8m0(min(127 + f - at, 254)), there ? 1.f : 0.f);
      if (lane == 0) {
        sh.meta[set].f = f + far;
        sh.meta[set].all = all;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.meta_full[set]);
    }
  } else if (warp >= W_DEQ) {
    // ------------------------------------------------------------ codes to operands
    reg_dec<R_DEQ>();
    const int x = tid - W_DEQ * 32;  // 0 .. 127
    constexpr int LR = D / 16, KP = D / 32, KR = 128 / LR;  // 16-byte pieces of a row, pieces a thread, rows apart
    constexpr int VB = D == 32 ? 4 : D / 16;                // bytes of a value row a thread transposes
    constexpr int VL = D / VB, VW = VB / 4;                 // lanes a value row
    for (int j = 0; j < steps; ++j) {
      const int st = j & 1;
      const uint32_t ph = (j >> 1) & 1;
      const uint32_t raw = base + L::R_OFF + j % RAW * L::R_BYTES;
      if (!wait(&sh.raw_full[j % RAW], (j / RAW) & 1) || !wait(&sh.k_empty[st], ph ^ 1u)) break;
      uint8_t *kt = smem + L::K_OFF + st * L::K_BYTES;
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        const int tok = i * KR + x / LR, c = x % LR;
        uint32_t w[4];
        shared_words<16>(raw + i * 2048 + x * 16, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] ^= 0x80808080u;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<uint4 *>(kt + L::chunk(c, h) * L::K_LBO + tok / 8 * 128 + tok % 8 * 16) =
              make_uint4(half_lo(w[2 * h]), half_hi(w[2 * h]), half_lo(w[2 * h + 1]), half_hi(w[2 * h + 1]));
      }
      tc::fence_proxy_async_smem();
      mbar_arrive(&sh.k_full[st]);
      if (!wait(&sh.v_empty[st], ph ^ 1u)) break;
      if (x < 8 * VL) {
        uint32_t y[8][VW];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          shared_words<VB>(raw + NT * D + (x / VL * 8 + i) * D + x % VL * VB, y[i]);
#pragma unroll
          for (int w = 0; w < VW; ++w) y[i][w] ^= 0x80808080u;
        }
        uint8_t *vt = smem + L::V_OFF + st * L::V_BYTES + x / VL * L::V_LBO;
#pragma unroll
        for (int w = 0; w < VW; ++w) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // elements 2 h and 2 h + 1 of the word, tokens in pairs
            uint32_t z[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = prmt(y[2 * i][w], y[2 * i + 1][w], h ? 0x7362 : 0x5140);
            const int d = x % VL * VB + 4 * w + 2 * h;
            uint8_t *dst = vt + d / 8 * L::V_SBO + d % 8 * 16;
            *reinterpret_cast<uint4 *>(dst) = make_uint4(half_lo(z[0]), half_lo(z[1]), half_lo(z[2]), half_lo(z[3]));
            *reinterpret_cast<uint4 *>(dst + 16) = make_uint4(half_hi(z[0]), half_hi(z[1]), half_hi(z[2]), half_hi(z[3]));
          }
        }
      }
      tc::fence_proxy_async_smem();
      mbar_arrive(&sh.v_full[st]);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.raw_empty[j % RAW]);
    }
  } else if (warp < 4 * L::RT) {
    // ------------------------------------------------------------ rows
    reg_inc<R_ROWS>();
    const int i = warp >> 2, rho = rho0 + i * TILE + (tid & (TILE - 1)), first = rho - lane;  // first: the warp's first row
    const uint32_t quad = (uint32_t)(warp & 3) << 21;  // this warp's 32 lanes of tensor memory
    const int p = row_pos(a, s, rho);
    const int p_min = __reduce_min_sync(0xffffffffu, p), p_max = __reduce_max_sync(0xffffffffu, p);
    // rows of q and out: LR lanes of 16 bytes (E elements) a row, RI rows an instruction
    constexpr int E = 16 / (int)sizeof(T), LR = D / E, RI = 32 / LR;
    uint8_t *mine = smem + i * L::QP * L::Q_BYTES;  // the row tile's query operand, at the end its output rows
    float rowf = 0.f;
#pragma unroll
    for (int x0 = 0; x0 < 32 / RI; x0 += 8) {
      constexpr int B = 32 / RI < 8 ? 32 / RI : 8;  // instructions in flight
      uint4 raw[B];
#pragma unroll
      for (int x = 0; x < B; ++x) {
        const int row = min(first + (x0 + x) * RI + lane / LR, s.n * a.G - 1);
        raw[x] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (s.r0 + row / a.G) * a.ld +
                                                  (size_t)(kvh * a.G + row % a.G) * D + lane % LR * E);
      }
#pragma unroll
      for (int x = 0; x < B; ++x) {
        float y[E], amax = 0.f;
        load4<T>(reinterpret_cast<const T *>(&raw[x]), reinterpret_cast<float(&)[4]>(y[0]));
        if constexpr (E == 8) load4<T>(reinterpret_cast<const T *>(&raw[x]) + 4, reinterpret_cast<float(&)[4]>(y[4]));
#pragma unroll
        for (int e = 0; e < E; ++e) amax = y[e] == y[e] ? fmaxf(amax, fabsf(y[e])) : INFINITY;
#pragma unroll
        for (int d = 1; d < LR; d *= 2) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
        const float up = fp16_range(amax), back = __shfl_sync(0xffffffffu, a.scale_log2 / up, lane % RI * LR);
        if (lane / RI == x0 + x) rowf = back;
        uint32_t hi[E / 2], lo[E / 2];
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          const float y0 = y[2 * e] * up, y1 = y[2 * e + 1] * up;
          hi[e] = pack_half(y0, y1);
          if (L::QP == 2) lo[e] = pack_rest(y0, y1, hi[e]);
        }
        const int r = (warp & 3) * 32 + (x0 + x) * RI + lane / LR, d = lane % LR * E;
        uint8_t *dst = mine + L::chunk(d / 16, d / 8 % 2) * L::Q_LBO + r / 8 * 128 + r % 8 * 16 + d % 8 * 2;
        if constexpr (E == 8) {
          *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        } else {
          *reinterpret_cast<uint2 *>(dst) = make_uint2(hi[0], hi[1]);
          *reinterpret_cast<uint2 *>(dst + L::Q_BYTES) = make_uint2(lo[0], lo[1]);
        }
        if constexpr (E == 8 && L::QP == 2) static_assert(E == 4, "two query pieces are fp32's");
      }
    }
    tc::fence_proxy_async_smem();
    mbar_arrive(&sh.q_full);
    auto total = [&]() {  // this row's place (a row that fills up the tile has none)
      return a.total + ((size_t)(s.r0 + rho / a.G) * a.H + kvh * a.G + rho % a.G) * total_row(D);
    };
    float m = LOWEST;
    uint64_t ls[2] = {0, 0};  // the sum l, in four parts
    int f = 0;
    bool ok = true;
    for (int j = 0; j < steps; ++j) {
      const int st = j & 1, set = j / META & 1;
      if (j % META == 0) ok = wait(&sh.meta_full[set], j / META >> 1 & 1);
      ok = ok && wait(&sh.s_full[i][st], (j >> 1) & 1);
      if (!ok) break;
      tc::fence_after_sync();
      uint32_t sv[4][16];
#pragma unroll
      for (int g = 0; g < 4; ++g) tc::ld16(s_col(i, st) + quad + 16 * g, sv[g]);
      tc::wait_ld();
#pragma unroll
      for (int g = 0; g < 4; ++g) tc::loaded16(sv[g]);
      const Scales &meta = sh.meta[set];
      const float4 *scale_of = meta.g[j % META];
      const int pos0 = (t0 + j) * NT;
      const bool inside = pos0 + NT - 1 <= p_min && (a.window <= 0 || pos0 > p_max - a.window) && meta.all;
      float mg[4], back[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 e = scale_of[g];
        back[g] = e.z;
        const uint64_t c = pair(rowf * e.x, rowf * e.x), d = pair(e.y, e.y);
#pragma unroll
        for (int k = 0; k < 16; k += 2) split(fma2(pair(u2f(sv[g][k]), u2f(sv[g][k + 1])), c, d), sv[g][k], sv[g][k + 1]);
      }
      if (!inside) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int at = pos0 + 16 * g + k;
            if (!(at <= p && (a.window <= 0 || at > p - a.window) && scale_of[g].w != 0.f)) sv[g][k] = __float_as_uint(-INFINITY);
          }
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float m0 = u2f(sv[g][0]), m1 = u2f(sv[g][1]);
#pragma unroll
        for (int k = 2; k < 16; k += 4) {
          m0 = fmaxf(fmaxf(m0, u2f(sv[g][k])), u2f(sv[g][k + 1]));
          if (k + 2 < 16) m1 = fmaxf(fmaxf(m1, u2f(sv[g][k + 2])), u2f(sv[g][k + 3]));
        }
        mg[g] = fmaxf(m0, m1);
      }
      const float mx = fmaxf(fmaxf(mg[0], mg[1]), fmaxf(mg[2], mg[3]));
      // a larger f scales l; from 0, after blocks of zeros, it also moves M (kv8_attention.cu: raise)
      if (meta.f > f) {
        if (j > 0) {
          const float by = (float)max(0, meta.f - f - FAR), w = ex2((float)(meta.f - f) - by);
          if (m > LOWEST) m += by;
          ls[0] = mul2(ls[0], pair(w, w));
          ls[1] = mul2(ls[1], pair(w, w));
        }
        f = meta.f;
      }
      const bool rise = __any_sync(0xffffffffu, mx - m > SLACK);
      const bool fold = TOTAL && j > 0 && (j & anew) == 0;
      if (rise || fold || (L::FOLD && j > 0)) {
        float scale = 1.f;
        if (rise) {
          const float to = fmaxf(m, reference(mx, HEAD, SLACK));
          scale = ex2(m - to);
          m = to;
          ls[0] = mul2(ls[0], pair(scale, scale));
          ls[1] = mul2(ls[1], pair(scale, scale));
        }
        if (j > 0) {
          ok = wait(&sh.pv_done[i][st ^ 1], ((j - 1) >> 1) & 1);
          if (!ok) break;
          tc::fence_after_sync();
          if (TOTAL && fold) {
            add_total<D>(total(), rho < s.n * a.G, j > anew + 1LL, m, [&](int c, uint32_t (&o)[16]) {
              tc::ld16(o_col(i) + quad + c, o);
              tc::wait_ld();
              tc::loaded16(o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(u2f(o[k]) * scale);
            });
          } else {
#pragma unroll
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16], t[16];
              const bool both = L::FOLD && j > 1;
              tc::ld16(o_col(i) + quad + c, o);
              if (both) tc::ld16(t_col(i) + quad + c, t);
              tc::wait_ld();
              tc::loaded16(o);
              if (both) tc::loaded16(t);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint((both ? u2f(t[k]) + u2f(o[k]) : u2f(o[k])) * scale);
              tc::st16((L::FOLD ? t_col(i) : o_col(i)) + quad + c, o);
            }
          }
        }
      }
      // weights, and P in the place of S
      const uint64_t less = pair(-m, -m);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const int g = 2 * half + k / 8, e = 2 * k % 16;
          uint32_t x0, x1;
          split(add2(pair(u2f(sv[g][e]), u2f(sv[g][e + 1])), less), x0, x1);
          const float w0 = ex2(u2f(x0)), w1 = ex2(u2f(x1));
          ls[k & 1] = fma2(pair(w0, w1), pair(back[g], back[g]), ls[k & 1]);
          hi[k] = pack_half(w0, w1);
          if (L::WP == 2) lo[k] = pack_rest(w0, w1, hi[k]);
        }
        tc::st16(s_col(i, st) + quad + 16 * half, hi);
        if (L::WP == 2) tc::st16(s_col(i, st) + quad + NT / 2 + 16 * half, lo);
      }
      tc::wait_st();
      tc::fence_before_sync();
      mbar_arrive(&sh.p_full[i][st]);
      if (j % META == META - 1) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.meta_empty[set]);
      }
    }
    // all outputs are done (pv_done's last phase would not do: the one before may still be open)
    // (they follow every store of the query operand, in whose place the rows are staged; without a step a barrier
    // of the row tile's warps orders the two)
    if (steps == 0) named_bar_sync(1 + i, TILE);
    else if (ok) wait(&sh.fin, 0);
    tc::fence_after_sync();
    float l;
    {
      uint32_t x0, x1, x2, x3;
      split(ls[0], x0, x1);
      split(ls[1], x2, x3);
      l = (u2f(x0) + u2f(x1)) + (u2f(x2) + u2f(x3));
    }
    const float w = l == 0.f || steps == 0 ? 0.f : 1.f / l, top = pow2_e8m0(f);  // (2^f / l can be too small for fp32)
    // the warp's rows through shared memory (16-byte pieces change places by row), then out in whole rows
    T *stage = reinterpret_cast<T *>(mine) + (warp & 3) * 32 * D;
#pragma unroll
    for (int c = 0; c < D; c += 16) {
      uint32_t o[16];
      if (steps > 0) {
        uint32_t t[16];
        const bool both = L::FOLD && steps > 1;
        tc::ld16(o_col(i) + quad + c, o);
        if (both) tc::ld16(t_col(i) + quad + c, t);
        tc::wait_ld();
        tc::loaded16(o);
        if (both) tc::loaded16(t);
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (both) o[k] = __float_as_uint(u2f(o[k]) + u2f(t[k]));
        if (TOTAL && steps > anew + 1LL && rho < s.n * a.G) {
          const float *sum = total(), f = ex2(sum[D] - m);
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(fmaf(sum[c + k], f, u2f(o[k])));
        }
      }
#pragma unroll
      for (int k = 0; k < 16; k += E) {
        T *dst = stage + lane * D + (((c + k) / E ^ lane) & (LR - 1)) * E;
#pragma unroll
        for (int h = 0; h < E; h += 4) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = w == 0.f ? 0.f : u2f(o[k + h + e]) * w * top;
          store4<T>(dst + h, y);
        }
      }
    }
    __syncwarp();
#pragma unroll 4
    for (int x = 0; x < 32 / RI; ++x) {
      const int r = x * RI + lane / LR, row = first + r;
      const uint4 v = *reinterpret_cast<const uint4 *>(stage + r * D + ((lane % LR ^ r) & (LR - 1)) * E);
      if (row < s.n * a.G)
        *reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + ((size_t)(s.r0 + row / a.G) * a.H + kvh * a.G + row % a.G) * D +
                                   lane % LR * E) = v;
    }
    // the rows anew, one after another, where the scales lie too far apart (kv8_attn.cuh: FAR)
    if (steps > 0 && ok && f >= APART) {
      __syncwarp();  // behind the stores above
      const int lift = f > APART + 220 ? 20 : 0;
      for (int row = first; row < min(first + 32, s.n * a.G); ++row) {
        const size_t at = (size_t)(s.r0 + row / a.G);
        float m, l, o[D / 32];
        far_row<T, D>(a, b, kvh, static_cast<const T *>(a.q) + at * a.ld + (size_t)(kvh * a.G + row % a.G) * D,
                      __shfl_sync(0xffffffffu, p, row - first), 0, 0x7fffffff, lift, lane, m, l, o);
        T *dst = static_cast<T *>(a.out) + (at * a.H + kvh * a.G + row % a.G) * D + lane * (D / 32);
#pragma unroll
        for (int d = 0; d < D / 32; ++d) dst[d] = from_f<T>(l == 0.f ? 0.f : o[d] / l * (lift ? ex2((float)lift) : 1.f));
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == W_MMA) {
    tc::fence_after_sync();
    tc::dealloc(tmem, 512);
  }
}

template <typename T, int D, bool TOTAL>
void launch(const AttnArgs &a, cudaStream_t st) {
  constexpr int smem = Lay<T, D>::SMEM;
  static_assert(smem <= 227 * 1024, "operand tiles fit an SM's shared memory");
  static std::atomic<uint64_t> allowed{0};
  allow_smem(prompt_kernel<T, D, TOTAL>, smem, allowed);
  const unsigned tiles = (unsigned)(((long long)std::max(a.r.most, 1) * a.G + Lay<T, D>::ROWS - 1) / Lay<T, D>::ROWS);
  launch_chained(prompt_kernel<T, D, TOTAL>, dim3(a.c.KV, a.r.B, tiles), THREADS, smem, 1, st, a);
}
template <typename T, int D>
void launch(const AttnArgs &a, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (a.total) return launch<T, D, true>(a, st);
  }
  launch<T, D, false>(a, st);
}
template <typename T>
void launch(const AttnArgs &a, cudaStream_t st) {
  if (a.c.D == 32) launch<T, 32>(a, st);
  else if (a.c.D == 64) launch<T, 64>(a, st);
  else launch<T, 128>(a, st);
}

}  // namespace

int prompt_rows(int dtype, int D) { return dtype == LBC_F32 && D == 128 ? Lay<float, 128>::ROWS : 2 * TILE; }

void launch_prompt(const AttnArgs &a, int dtype, cudaStream_t st) {
  if (dtype == LBC_F32) launch<float>(a, st);
  else if (dtype == LBC_BF16) launch<__nv_bfloat16>(a, st);
  else launch<__half>(a, st);
}

}  // namespace kv8
}  // namespace lbc
