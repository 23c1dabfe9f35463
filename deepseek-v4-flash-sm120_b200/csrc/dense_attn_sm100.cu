// Dense causal attention over packed sequences with grouped heads (whole prompts, chunks of
// prompts behind a cached context, single tokens).
//
//   O_i = sum_j p_ij V_j / sum_j p_ij,   p_ij = exp(scale Q_i K_j),   j <= i + len_k - len_q
//
// One CTA owns two tiles of 128 query rows of one sequence and one group of heads, and walks
// the sequence's keys in tiles of 128.  A row is a (token, head) pair: the heads that share a
// key/value head are packed next to each other, so a single token of a group fills as much of
// a tile as it can, and a tile spans few tokens (little of it is masked).
//
//   S_s [128 rows, 128 keys] = Q_s K^T        A, B from shared memory, K-major
//   O_s [128 rows, d_v]     += P_s V          A = P from TMEM, B = V, MN-major as it was loaded
//
// A softmax thread owns one row (its TMEM lane), so the maximum and the sum of a row need no
// exchange.  It takes the 128 scores of a tile into registers at once and frees their TMEM
// columns: the two tiles (s = 0, 1) share one score buffer (O_0, O_1, P_0 and P_1 fill the rest
// of TMEM at d_v = 128), the scores of the next tile are formed while this one's exponentials
// are, and the product with V waits for neither.  O is rescaled
// only when a row's maximum has grown by more than 2^8 since its reference was set, by the same
// threads, so there is no correction stage.  The sums are 32-bit; P has as many significant bits
// at any scale in BF16, while FP16 weights are held 2^7 times as large (at most 2^15 then), which
// moves what FP16 cannot hold from 2^-25 of the reference's weight to 2^-32 (of 120000 keys 18 nats
// below another one, 0.2 % of the weight, nothing was left).  Q, K and V arrive by TMA; K's ring is
// recycled in blocks of 64 columns and V's in tiles, which is what the 227 KB allow at d_qk = 192.
//
// Masked keys: scores are replaced, not added to, so nothing in a masked key's K row counts.
// A product with weight zero would still let a NaN or an infinity of a masked V row through,
// so in the tiles that some row sees only in part an idle warp looks over V in shared memory
// before the tensor core may read it: rows no one sees are cleared, and elements that are not
// finite are cleared and handed by the epilogue to the rows that do see them.
//
// Few rows (single tokens over long contexts): the keys are cut into up to n_splits ranges, each
// CTA leaves normalised 32-bit partials, and dense_combine_kernel joins them.  A CTA whose
// second row tile would be empty then gives the first one's odd key tiles to the second
// pipeline ("twin"), which halves its chain of products and softmaxes; a range therefore has
// two partial sets.
//
// Measured.  One prompt of 8192, 16 heads, (192, 128), causal: 272 us from a cold clock, 1.26
// PFLOP/s of the products that are not masked (0.75 of a matrix product's rate), 328 us under the
// power limit; tensor pipe 64 % busy, bound by the 128 exponentials, sums and conversions of
// each thread and tile beside it.  Packed prompts, 24 heads on 4, (128, 128): 255 to 276 us from a
// cold clock, 302 under the power limit, tensor pipe 56 % busy: products and exponentials take equal
// clocks there and overlap in part, and an SM's ten CTAs start and end one after the other.  (64, 64),
// one prompt of 8192: 184 us, 119 of them for the exponentials alone.  Single tokens, 8 contexts of 1000
// to 16383, 32 heads on 8: 18 us a CTA for 99 MB, of which 13 us stream at memory's rate (with one
// unit of V less for twins 17) and 5 are its start and end; 31 us with the joining launch.
#include <cuda_fp16.h>

#include "attn_params.cuh"
#include "launch_util.h"
#include "launchers.h"
#include "sm100_ptx.cuh"
#include "tensor_map.h"

namespace dsv4 {

__device__ int g_dense_error = 0;

namespace {

using namespace ptx;

constexpr int TILE_M = 128, TILE_N = 128;
constexpr int BLOCK_BYTES = 128 * 128;               // [128 rows][64 16-bit values], swizzled
constexpr int SOFTMAX_THREADS = 256;                 // two warpgroups, one per row tile
constexpr int THREADS = SOFTMAX_THREADS + 128;       // + two MMA warps, TMA, looking over V
// 384 threads start with 168 registers; the third warpgroup hands most of its own over:
// 128 * 72 + 256 * 216 = 384 * 168.
constexpr int LAUNCH_REGS = 168, SOFTMAX_REGS = 216, HELPER_REGS = 72;
static_assert(SOFTMAX_THREADS * SOFTMAX_REGS + 128 * HELPER_REGS <= THREADS * LAUNCH_REGS,
              "setmaxnreg.inc can only take what setmaxnreg.dec gave back");
static_assert(THREADS * (LAUNCH_REGS + 8) > 65536, "LAUNCH_REGS is what the launch bound yields");
constexpr int WARP_QK = 8, WARP_PV = 9, WARP_TMA = 10, WARP_LOOK = 11;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float RESCALE_THRESHOLD = 8.0f;            // log2 units
constexpr float FP16_LIFT = 7.0f;                    // log2 of the factor on FP16 weights
constexpr uint32_t TMEM_COLS = 512;

enum DenseErr { ERR_Q = 11, ERR_K = 12, ERR_V = 13, ERR_P = 14, ERR_S = 15, ERR_O = 16, ERR_SLOT = 17, ERR_LOOK = 18,
                ERR_FREE = 19 };

template <int DQK, int DV> struct DCfg {
  static constexpr int QB = DQK / 64, VB = DV / 64;
  static constexpr int K_SLOTS = DQK == 192 ? 4 : DQK == 128 ? 6 : 4;   // blocks of 64 columns
  static constexpr int K_STEP = DQK == 192 ? 1 : QB;      // blocks handed over together
  static constexpr int K_RING = K_SLOTS / K_STEP;
  static constexpr int V_UNITS = DQK == 64 ? 4 : 2;                     // whole tiles; twins have one more
  // TMEM columns: O_s (d_v each), P_s (64 each), and what is left for scores: one tile that the
  // row tiles use in turn at d_v = 128, one each at d_v = 64.
  static constexpr int S_BUFS = DV == 64 ? 2 : 1;
  static constexpr uint32_t COL_S = 0, COL_P = 128 * S_BUFS, COL_O = COL_P + 128;
  static_assert(COL_O + 2 * DV <= TMEM_COLS, "512 columns");
  static_assert(V_UNITS <= 4 && VB <= QB, "a unit fits where the second Q tile would be");
  static constexpr int Q_BYTES = 2 * QB * BLOCK_BYTES, K_BYTES = K_SLOTS * BLOCK_BYTES;
  static constexpr int V_UNIT_BYTES = VB * BLOCK_BYTES, V_BYTES = V_UNITS * V_UNIT_BYTES;
};

// The part of a sequence that a CTA works on.
struct Work {
  int q0, len_q, k0, len_k;      // rows of the packed tensors
  int t0;                        // first query token of row tile 0, in the sequence
  int first, tiles;              // key tiles [first, first + tiles)
  int count[2];                  // of them row tile s takes the first count[s] ...
  bool twin;                     // ... or, both row tiles being the same, every second one from s on
  int look;                      // key tiles from this one on are seen only in part by some row
  bool any;
  int chunk, split;              // heads, range
  int last_set;                  // partial sets from here on are not written: this CTA marks them
};

struct DenseCtrl {
  uint64_t q_full[2], s_full[2], s_free[2], p_full[2], o_done[2];
  uint64_t k_full[4], k_empty[4], v_full[5], v_empty[5];
  // tiles that are looked over (the last ones) land on v_look instead of v_full, so that the
  // looking warps count only their own phases; v_clean hands them on
  uint64_t v_look[5], v_clean[5];
  uint32_t tmem;
  int fail, bad;
  Work work;                     // with ranges: what the loading warp has found
};

template <int DQK, int DV> constexpr size_t dense_smem_bytes() {
  using C = DCfg<DQK, DV>;
  return 1024 + C::Q_BYTES + C::K_BYTES + C::V_BYTES + sizeof(DenseCtrl);
}
static_assert(dense_smem_bytes<192, 128>() <= 232448 && dense_smem_bytes<128, 128>() <= 232448, "227 KB a CTA");

struct DenseParams {
  CUtensorMap mq, mk, mv;
  int b, t_q, t_k, h_q, h_kv, causal;
  int pack, tok_tile;            // heads packed per row tile, tokens per row tile
  int chunks;                    // head chunks: h_q / pack
  int slots;                     // row-tile pairs, upper bound over all sequences
  int n_splits;                  // ranges of a sequence's keys, at most
  int ctas;                      // of a launch with ranges
  int items;                     // row-tile pairs x head chunks, upper bound
  int sms;
  int sectors;                   // rows of the output start on 32 bytes
  float sm_scale;
  const int32_t *cu_q, *cu_k;
  const float* sink;
  const void* v;
  int64_t stride_v_t, stride_v_h, stride_o_t, stride_o_h, stride_ml_t, stride_lse_t;
  void* out;
  float *max_logits, *lse;
  float *o_accum, *stat_accum;   // [2 splits][t][h][d_v], [2 splits][t][h][2] (max logit, log-sum-exp)
};

// Pairs of 32-bit floats in one 64-bit register: one instruction for both.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// Largest of three; NaN if one of them is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF16) {
    __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&t);
  } else {
    __half2 t = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&t);
  }
}
// Which halves of a word are infinite or NaN (bits 15 and 31).
template <bool BF16>
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) {
  return BF16 ? ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u
              : ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}

// Larger magnitude in each half of a word (the sign is of no meaning); NaN if either is.
template <bool BF16>
__device__ __forceinline__ uint32_t abs_max2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (BF16) asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Keys of the sequence that token t sees: [0, reach).
__device__ __forceinline__ int reach_of(const DenseParams& p, const Work& w, int t) {
  if (!p.causal) return w.len_k;
  const int r = t + w.len_k - w.len_q + 1;
  return r < 0 ? 0 : r < w.len_k ? r : w.len_k;
}

__device__ __forceinline__ int clamp_to(int v, int lo, int hi) { return min(max(v, lo), hi); }

// Which tiles the rows from w.t0 on see of the keys' tiles [first, end).
template <bool RANGES>
__device__ __forceinline__ void set_tiles(const DenseParams& p, Work& w, int first, int end) {
  int tiles[2] = {0, 0};
  if (w.any) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int a = w.t0 + s * p.tok_tile;
      if (a < w.len_q)
        tiles[s] = (reach_of(p, w, min(a + p.tok_tile, w.len_q) - 1) + TILE_N - 1) / TILE_N;
    }
  }
  const int total = max(tiles[0], tiles[1]);
  w.first = min(first, total);
  end = min(end, total);
  w.tiles = end - w.first;
#pragma unroll
  for (int s = 0; s < 2; ++s) w.count[s] = max(min(tiles[s], end) - w.first, 0);
  w.twin = RANGES && w.t0 + p.tok_tile >= w.len_q;
  if (w.twin) {
    w.count[0] = (w.tiles + 1) / 2;
    w.count[1] = w.tiles / 2;
  }
  w.look = reach_of(p, w, w.t0) / TILE_N;
}

__device__ __forceinline__ Work find_work(const DenseParams& p, int block) {
  Work w;
  // Slots last to first: in a causal sequence the late rows are the long ones.
  w.chunk = block % p.chunks;
  const int slot = p.slots - 1 - block / p.chunks;
  w.split = w.last_set = 0;
  // Sequence s owns the slots from cu_q[s] / span + s on: at least ceil(len / span) of them.
  // Every warp looks for it 32 candidates at a time: the loads of a step do not wait for one
  // another (bisection took one memory latency a halving, up to 2 us of a short CTA's 8).
  const int span = 2 * p.tok_tile, lane = threadIdx.x & 31;
  int lo = 0, n = p.b;                     // the sequence is one of [lo, lo + n)
  int q0, q1, k0, k1;
  if (n < 32) {                            // all bounds at once
    const int cq = __ldg(p.cu_q + min(lane, n)), ck = __ldg(p.cu_k + min(lane, n));
    const bool below = lane < n && clamp_to(cq, 0, p.t_q) / span + lane <= slot;
    lo = 31 - __clz(__ballot_sync(0xffffffffu, below) | 1u);
    q0 = __shfl_sync(0xffffffffu, cq, lo);
    q1 = __shfl_sync(0xffffffffu, cq, lo + 1);
    k0 = __shfl_sync(0xffffffffu, ck, lo);
    k1 = __shfl_sync(0xffffffffu, ck, lo + 1);
    n = 0;
  }
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lo + lane * step;
    const bool below = lane * step < n && clamp_to(__ldg(p.cu_q + at), 0, p.t_q) / span + at <= slot;
    const uint32_t hits = __ballot_sync(0xffffffffu, below) | 1u;
    const int last = 31 - __clz(hits);     // (bounds that do not ascend land somewhere, in range)
    n = min(step, n - last * step);
    lo += last * step;
  }
  if (n > 0) {
    q0 = __ldg(p.cu_q + lo), q1 = __ldg(p.cu_q + lo + 1), k0 = __ldg(p.cu_k + lo), k1 = __ldg(p.cu_k + lo + 1);
  }
  w.q0 = clamp_to(q0, 0, p.t_q);
  w.len_q = clamp_to(q1, w.q0, p.t_q) - w.q0;
  w.k0 = clamp_to(k0, 0, p.t_k);
  w.len_k = clamp_to(k1, w.k0, p.t_k) - w.k0;
  const int64_t t0 = static_cast<int64_t>(slot - (w.q0 / span + lo)) * span;
  w.any = t0 >= 0 && t0 < w.len_q;
  w.t0 = static_cast<int>(w.any ? t0 : 0);
  set_tiles<false>(p, w, 0, 0x7fffffff);
  return w;
}

__device__ __forceinline__ float root(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// With ranges: the sequences are cut into ranges of about the same length, so that the grid ends
// evenly whatever their lengths: the shortest length with which the launch's CTAs are enough (and
// they are for line / (ctas - items) tiles, line being the sum of all items' tiles, since rounding
// up costs every item less than one range more).  A range streams a tile in about 1 us and costs
// 0.6 us to start and join, so below sqrt(0.6 tiles) shorter ranges gain nothing.  (As many ranges
// for every sequence instead, microseconds: 8 of 1000 to 16383 keys, 32 heads on 8, 5 query tokens
// each: 47, with this 35; 60 of 1 to 20000 keys, 8 heads of 64: 170 uncut and 100 in two, with this 80.)
__device__ __forceinline__ Work find_range(const DenseParams& p, int block) {
  Work w = {};
  const int span = 2 * p.tok_tile, lane = threadIdx.x & 31;
  int q0 = 0, len_q = 0, k0 = 0, len_k = 0;             // of sequence s0 + lane
  int items = 0, tiles = 0, shortest = 1;               // its row-tile pairs x chunks, key tiles, shortest range
  auto fetch = [&](int s0) {
    const int s = min(s0 + lane, p.b - 1);
    const int a = __ldg(p.cu_q + s), b = __ldg(p.cu_q + s + 1), c = __ldg(p.cu_k + s), d = __ldg(p.cu_k + s + 1);
    q0 = clamp_to(a, 0, p.t_q);
    len_q = s0 + lane < p.b ? clamp_to(b, q0, p.t_q) - q0 : 0;
    k0 = clamp_to(c, 0, p.t_k);
    len_k = clamp_to(d, k0, p.t_k) - k0;
    items = (len_q + span - 1) / span * p.chunks;
    tiles = (len_k + TILE_N - 1) / TILE_N;
    shortest = max(static_cast<int>(ceilf(root(0.6f * tiles))), 1);
  };
  // ceil(tiles / per), or a little less beyond 2^18 tiles, but never more: the factor outweighs what
  // the quick division can be off
  auto parts_of = [&](int even) {
    const int per = max(even, shortest);
    return clamp_to(static_cast<int>(__fdividef(tiles + (per - 0.5f), per) * (1.f - 0x1p-20f)), 1, p.n_splits);
  };
  // the line's length in floating point (64-bit divisions took a third of the time), rounded up so
  // that `even` is never too short
  float line = 0.f;
  for (int s0 = 0; s0 < p.b; s0 += 32) {
    fetch(s0);
    line = __fmaf_ru(static_cast<float>(items), static_cast<float>(tiles), line);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) line = __fadd_ru(line, __shfl_xor_sync(0xffffffffu, line, d));
  // no shorter than an SM's share of the line: that would only add starts
  int low = static_cast<int>(fminf(ceilf(line / p.sms), 0x1p24f));
  int even = max(static_cast<int>(fminf(ceilf(__fdiv_ru(line, p.ctas - p.items)), 0x1p24f)), low);
  while (low < even) {                                  // (only with fewer items than SMs; few steps)
    const int mid = (low + even) / 2;
    uint32_t count = 0;
    for (int s0 = 0; s0 < p.b; s0 += 32) {
      if (p.b > 32) fetch(s0);
      count += min(static_cast<uint32_t>(items * parts_of(mid)), static_cast<uint32_t>(p.ctas) + 1);
    }
    if (__reduce_add_sync(0xffffffffu, count) <= static_cast<uint32_t>(p.ctas)) even = mid;
    else low = mid + 1;
  }
  uint32_t before = 0;                                  // CTAs of the sequences before s0
  w.any = false;
  for (int s0 = 0; s0 < p.b && !w.any; s0 += 32) {
    if (p.b > 32) fetch(s0);
    const int parts = parts_of(even), per = (tiles + parts - 1) / parts;
    const uint32_t mine = min(static_cast<uint32_t>(items * parts), static_cast<uint32_t>(p.ctas));
    uint32_t sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, before + sum > static_cast<uint32_t>(block));
    if (hit != 0) {
      const int from = __ffs(hit) - 1;
      const int r = block - static_cast<int>(before + __shfl_sync(0xffffffffu, sum - mine, from));
      const int n = __shfl_sync(0xffffffffu, parts, from), len = __shfl_sync(0xffffffffu, per, from);
      w.q0 = __shfl_sync(0xffffffffu, q0, from);
      w.len_q = __shfl_sync(0xffffffffu, len_q, from);
      w.k0 = __shfl_sync(0xffffffffu, k0, from);
      w.len_k = __shfl_sync(0xffffffffu, len_k, from);
      w.split = r % n;
      w.chunk = r / n % p.chunks;
      w.t0 = r / n / p.chunks * span;
      w.last_set = w.split == n - 1 ? 2 * n : 2 * p.n_splits;
      w.any = true;
      set_tiles<true>(p, w, w.split * len, w.split * len + len);
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return w;
}

// Where a row's results go, and its final factor.
__device__ __forceinline__ void store_stats(const DenseParams& p, int set, int64_t t, int h, float m_raw, float m_ref,
                                            float l, bool fail, float& factor) {
  // m_ref: reference in log2 units (-inf: nothing seen); l: sum relative to it
  const bool none = m_ref == -INFINITY && l == l;      // (NaN scores set no reference, but show)
  const float lse = none ? -INFINITY : logf(l) + m_ref * LN2;
  const float ml = none ? -INFINITY : m_raw * p.sm_scale;
  factor = none ? 0.f : 1.f / l;
  if (p.n_splits > 1) {
    float2* dst = reinterpret_cast<float2*>(p.stat_accum + ((static_cast<int64_t>(set) * p.t_q + t) * p.h_q + h) * 2);
    *dst = make_float2(ml, fail ? NAN : lse);
    return;
  }
  if (p.sink != nullptr && !none) factor *= 1.f / (1.f + expf(p.sink[h] - lse));
  p.max_logits[t * p.stride_ml_t + h] = ml;
  p.lse[t * p.stride_lse_t + h] = fail ? NAN : none ? INFINITY : lse;
}

// RANGES: the keys are cut into n_splits ranges, with twins (an instantiation of its own: the
// choice inside the loops costs 4 to 6 % of a long prompt).
template <int DQK, int DV, bool BF16, bool RANGES>
__global__ void __launch_bounds__(THREADS, 1)
dense_attn_kernel(const __grid_constant__ DenseParams p) {
  using C = DCfg<DQK, DV>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t sQ = base, sK = sQ + C::Q_BYTES, sV = sK + C::K_BYTES;
  DenseCtrl& ctrl = *reinterpret_cast<DenseCtrl*>(smem_raw + (base - raw) + C::Q_BYTES + C::K_BYTES + C::V_BYTES);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto bar = [&](uint64_t* x) { return smem_u32(x); };
  if (warp == WARP_LOOK) {      // (the warp that has nothing to do at the start)
    if (lane == 0) {
      for (int s = 0; s < 2; ++s) {
        mbar_init(bar(&ctrl.q_full[s]), 1);
        mbar_init(bar(&ctrl.s_full[s]), 1);
        mbar_init(bar(&ctrl.s_free[s]), 4);
        mbar_init(bar(&ctrl.p_full[s]), 4);
        mbar_init(bar(&ctrl.o_done[s]), 1);
      }
      for (int i = 0; i < 4; ++i) {
        mbar_init(bar(&ctrl.k_full[i]), 1);
        mbar_init(bar(&ctrl.k_empty[i]), 1);
      }
      for (int i = 0; i < 5; ++i) {
        mbar_init(bar(&ctrl.v_full[i]), 1);
        mbar_init(bar(&ctrl.v_empty[i]), 1);
        mbar_init(bar(&ctrl.v_look[i]), 1);
        mbar_init(bar(&ctrl.v_clean[i]), 1);
      }
      ctrl.fail = 0;
      ctrl.bad = 0;
      mbar_init_fence();
    }
    __syncwarp();
    tmem_alloc(smem_u32(&ctrl.tmem), TMEM_COLS);
    tmem_relinquish();
  } else if (warp == WARP_TMA && lane < 3) {
    tma_prefetch_map(lane == 0 ? &p.mq : lane == 1 ? &p.mk : &p.mv);
  }
  grid_dependency_wait();
  Work w;
  if constexpr (RANGES) {          // one warp looks: twelve would share four schedulers
    if (warp == WARP_TMA) {
      w = find_range(p, blockIdx.x);
      if (lane == 0) ctrl.work = w;
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    w = ctrl.work;
  } else {
    w = find_work(p, blockIdx.x);
  }
  const bool twin = RANGES && w.twin;
  // twins share a Q tile; in the place of the second one they have one more unit of V
  const int v_units = twin ? C::V_UNITS + 1 : C::V_UNITS;
  auto v_at = [&](int vu) { return RANGES && vu == C::V_UNITS ? sQ + C::QB * BLOCK_BYTES : sV + vu * C::V_UNIT_BYTES; };
  auto give_back = [&]() {                // TMEM of a CTA that leaves before the others have seen it
    if (warp != WARP_LOOK) return;
    tc_fence_before_sync();
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(*reinterpret_cast<volatile uint32_t*>(&ctrl.tmem), TMEM_COLS);
  };
  if (!w.any) {
    give_back();
    return;
  }
  const int head0 = w.chunk * p.pack;
  const int kvh = head0 / (p.h_q / p.h_kv);
  const int n_tiles = w.tiles;

  if (n_tiles == 0) {                     // nothing in this CTA's range: results of empty rows
    const int rows = 2 * p.tok_tile * p.pack;
    for (int i = tid; i < rows; i += THREADS) {
      const int tok = w.t0 + i / p.pack, h = head0 + i % p.pack;
      if (tok >= w.len_q) continue;
      const int64_t t = w.q0 + tok;
      float f;
      if (RANGES) {                       // (a set without weight: its values are not read)
        for (int set = 2 * w.split; set < 2 * w.split + 2; ++set) store_stats(p, set, t, h, -INFINITY, -INFINITY, 0.f, false, f);
        for (int set = w.last_set; set < 2 * p.n_splits; ++set) store_stats(p, set, t, h, -INFINITY, -INFINITY, 0.f, false, f);
      } else {
        store_stats(p, 0, t, h, -INFINITY, -INFINITY, 0.f, false, f);
        uint4* d = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + t * p.stride_o_t + h * p.stride_o_h);
        for (int c = 0; c < DV / 8; ++c) d[c] = make_uint4(0, 0, 0, 0);
      }
    }
    give_back();
    return;
  }

  if (!RANGES) {
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
  }
  const uint32_t tmem = ctrl.tmem;
  // A lane whose bounded wait gives up records it, waits for nothing any more and issues nothing; but
  // it walks on through the same loops, so that its warp stays together for what the whole warp has
  // to execute (a phase may complete just as the first lanes give up).  The other roles then run into
  // their own limits, long after every copy and product in flight has finished.
  auto gave_up = [&](int code) {
    atomicExch(&g_dense_error, code);
    *reinterpret_cast<volatile int*>(&ctrl.fail) = 1;
  };

  if (warp >= WARP_QK) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(HELPER_REGS));
    if (warp == WARP_TMA) {
      // ======================= loads ======================================================
      if (elect_one()) {
        const uint32_t q_bytes = static_cast<uint32_t>(p.pack * p.tok_tile) * 128u;
        auto load_q = [&](int s) {
          mbar_expect_tx(bar(&ctrl.q_full[s]), q_bytes * C::QB);
          for (int c = 0; c < C::QB; ++c)
            tma_load_3d(sQ + (s * C::QB + c) * BLOCK_BYTES, &p.mq, 64 * c, head0,
                        w.q0 + w.t0 + s * p.tok_tile, bar(&ctrl.q_full[s]));
        };
        if (w.count[0] > 0) load_q(0);
        bool ok = true;                  // (one lane alone: it may stop)
        int ks = 0, kphase = 0, vu = 0, vphase = 0;
        auto wait = [&](uint64_t* b, int parity) {
          if (ok && !mbar_wait_fast(bar(b), parity)) {
            gave_up(ERR_SLOT);
            ok = false;
          }
          return ok;
        };
        for (int i = 0; i < n_tiles; ++i) {
          const int row = w.k0 + (w.first + i) * TILE_N;
          for (int c = 0; c < C::QB; c += C::K_STEP) {
            if (!wait(&ctrl.k_empty[ks], kphase ^ 1)) break;
            mbar_expect_tx(bar(&ctrl.k_full[ks]), C::K_STEP * BLOCK_BYTES);
            for (int d = 0; d < C::K_STEP; ++d)
              tma_load_3d(sK + (ks * C::K_STEP + d) * BLOCK_BYTES, &p.mk, 64 * (c + d), kvh, row, bar(&ctrl.k_full[ks]));
            if (++ks == C::K_RING) { ks = 0; kphase ^= 1; }
          }
          if (i == 0 && w.count[1] > 0 && !twin) load_q(1);
          if (!wait(&ctrl.v_empty[vu], vphase ^ 1)) break;
          const uint32_t landed = bar(w.first + i >= w.look ? &ctrl.v_look[vu] : &ctrl.v_full[vu]);
          mbar_expect_tx(landed, C::V_UNIT_BYTES);
          for (int c = 0; c < C::VB; ++c)
            tma_load_3d(v_at(vu) + c * BLOCK_BYTES, &p.mv, 64 * c, kvh, row, landed);
          if (++vu == v_units) { vu = 0; vphase ^= 1; }
        }
      }
      __syncwarp();
    } else if (warp < WARP_TMA) {
      // ======================= products ===================================================
      // One warp issues the scores of both row tiles, another one the products with V: the two
      // streams write different accumulators and interleave in the tensor core, and a wait of
      // one does not hold up the other.  Every lane runs the code, one issues; the values it
      // starts from are broadcast so that they are known to be uniform.
      const uint32_t t0 = __shfl_sync(0xffffffffu, tmem, 0);
      const int count0 = __shfl_sync(0xffffffffu, w.count[0], 0), count1 = __shfl_sync(0xffffffffu, w.count[1], 0);
      const int tiles = __shfl_sync(0xffffffffu, w.tiles, 0);
      const bool twin = RANGES && __shfl_sync(0xffffffffu, w.twin ? 1 : 0, 0) != 0;
      // does row tile s read key tile i, and as its how manieth?
      auto takes = [&](int s, int i) { return twin ? (i & 1) == s : i < (s == 0 ? count0 : count1); };
      auto nth = [&](int i) { return twin ? i >> 1 : i; };
      const uint32_t elected = elect_one();
      bool ok = true;
      auto wait = [&](uint64_t* b, int parity, int code) {
        if (ok && !mbar_wait_fast(bar(b), parity)) {
          if (elected) gave_up(code);
          ok = false;
        }
      };                                 // (no lane needs another one here; a __syncwarp took 0.6 % more)
      if (warp == WARP_QK) {
        constexpr uint32_t idesc = make_idesc_16(BF16, TILE_M, TILE_N, 0, 0);
        const uint64_t dQ = make_smem_desc(sQ, 16, 1024, SWZ_128B);
        const uint64_t dK = make_smem_desc(sK, 16, 1024, SWZ_128B);
        int turn = 0;                                    // score tiles so far
#pragma unroll 1
        for (int i = 0; i < tiles; ++i) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (!takes(s, i)) continue;
            const bool last = twin || s == 1 || i >= count1;     // nobody reads the tile's K after this
            const int j = nth(i);
            if (j == 0) wait(&ctrl.q_full[twin ? 0 : s], 0, ERR_Q);
            // the scores that were here have been read
            if (C::S_BUFS == 1) wait(&ctrl.s_free[0], (turn & 1) ^ 1, ERR_FREE);
            else wait(&ctrl.s_free[s], (j & 1) ^ 1, ERR_FREE);
            ++turn;
            const uint32_t tS = t0 + C::COL_S + (C::S_BUFS == 1 ? 0 : 128 * s);
            int ks = (i * (C::QB / C::K_STEP)) % C::K_RING, kphase = (i * (C::QB / C::K_STEP) / C::K_RING) & 1;
#pragma unroll
            for (int c = 0; c < C::QB; c += C::K_STEP) {
              wait(&ctrl.k_full[ks], kphase, ERR_K);
              tc_fence_after_sync();
              const uint64_t d = dK + ((ks * C::K_STEP * BLOCK_BYTES) >> 4);
              if (ok) {
#pragma unroll
                for (int k = 0; k < 4 * C::K_STEP; ++k)
                  umma_bf16_elect(tS, dQ + ((((twin ? 0 : s) * C::QB + c + (k >> 2)) * BLOCK_BYTES + (k & 3) * 32) >> 4),
                                  d + (((k >> 2) * BLOCK_BYTES + (k & 3) * 32) >> 4), idesc, (c | k) != 0, elected);
                if (last) umma_commit_elect(bar(&ctrl.k_empty[ks]), elected);
              }
              if (++ks == C::K_RING) { ks = 0; kphase ^= 1; }
            }
            if (ok) umma_commit_elect(bar(&ctrl.s_full[s]), elected);
          }
        }
      } else {
        constexpr uint32_t idesc = make_idesc_16(BF16, TILE_M, DV, 0, 1);
        const uint64_t dV = make_smem_desc(sV, BLOCK_BYTES, 1024, SWZ_128B);   // MN-major
        const uint64_t dV_more = make_smem_desc(sQ + C::QB * BLOCK_BYTES, BLOCK_BYTES, 1024, SWZ_128B);
        const int units = twin ? C::V_UNITS + 1 : C::V_UNITS;
        uint32_t clean_parity = 0;
#pragma unroll 1
        for (int i = 0; i < tiles; ++i) {
          const int vu = i % units, vphase = (i / units) & 1;
          const uint64_t d = RANGES && vu == C::V_UNITS ? dV_more : dV + ((vu * C::V_UNIT_BYTES) >> 4);
          if (w.first + i >= w.look) {
            wait(&ctrl.v_clean[vu], (clean_parity >> vu) & 1, ERR_LOOK);
            clean_parity ^= 1u << vu;
          } else {
            wait(&ctrl.v_full[vu], vphase, ERR_V);
          }
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (!takes(s, i)) continue;
            const int j = nth(i);
            wait(&ctrl.p_full[s], j & 1, ERR_P);
            tc_fence_after_sync();
            if (!ok) continue;
#pragma unroll
            for (int k = 0; k < TILE_N / 16; ++k)
              umma_ts_elect(t0 + C::COL_O + DV * s, t0 + C::COL_P + 64 * s + 8 * k, d + ((k * 2048) >> 4), idesc,
                            (j | k) != 0, elected);
            umma_commit_elect(bar(&ctrl.o_done[s]), elected);
            if (twin || s == 1 || i >= count1) umma_commit_elect(bar(&ctrl.v_empty[vu]), elected);
          }
        }
      }
    } else {
      // ======================= looking over V =============================================
      // keys the whole CTA sees (its last row sees the most)
      const int seen = reach_of(p, w, min(w.t0 + 2 * p.tok_tile, w.len_q) - 1);
      uint32_t parity = 0;
      bool ok = true;
      for (int i = max(w.look - w.first, 0); i < n_tiles; ++i) {
        const int vu = i % v_units;
        if (ok && !mbar_wait_fast(bar(&ctrl.v_look[vu]), (parity >> vu) & 1)) {
          gave_up(ERR_V);
          ok = false;
        }
        __syncwarp();
        parity ^= 1u << vu;
        const int live = min(seen - (w.first + i) * TILE_N, TILE_N);   // rows of the tile that count
        // 32 chunks of 16 bytes (four rows of a block) at a time
        constexpr int BATCH = 8;
        const uint32_t mine = v_at(vu) + lane * 16;
        uint32_t most = 0;                           // largest magnitude, pairwise; NaN stays
        for (int c0 = 0; c0 < C::V_UNIT_BYTES / 512; c0 += BATCH) {
          uint32_t x[BATCH][4];
#pragma unroll
          for (int k = 0; k < BATCH; ++k) {
            const int row = ((c0 + k) * 4 + (lane >> 3)) & 127;
            const uint32_t addr = mine + (c0 + k) * 512;
            x[k][0] = x[k][1] = x[k][2] = x[k][3] = 0;
            if (row < live)
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(x[k][0]), "=r"(x[k][1]), "=r"(x[k][2]), "=r"(x[k][3]) : "r"(addr) : "memory");
            else
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(addr), "r"(0) : "memory");
          }
#pragma unroll
          for (int k = 0; k < BATCH; ++k)
#pragma unroll
            for (int q = 0; q < 4; ++q) most = abs_max2<BF16>(most, x[k][q]);
        }
        const bool found = not_finite2<BF16>(most) != 0;
        if (found) {                                 // rare: clear them
          for (int c = 0; c < C::V_UNIT_BYTES / 512; ++c) {
            const uint32_t addr = mine + c * 512;
            uint32_t x[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(addr) : "memory");
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t h = not_finite2<BF16>(x[q]);
              if (h & 0x8000u) x[q] &= 0xffff0000u;
              if (h & 0x80000000u) x[q] &= 0x0000ffffu;
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                         ::"r"(addr), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
          }
        }
        if (found) *reinterpret_cast<volatile int*>(&ctrl.bad) = 1;
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(&ctrl.v_clean[vu]));
      }
    }
    grid_launch_dependents();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == WARP_LOOK) tmem_dealloc(tmem, TMEM_COLS);
    return;
  }

  // ======================= softmax ======================================================
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
  const int s = warp >> 2;
  const int row = (warp & 3) * 32 + lane;
  const int row_t0 = w.t0 + (twin ? 0 : s * p.tok_tile);
  const int tok = row_t0 + row / p.pack;
  const int h = head0 + row % p.pack;
  const bool live = row < p.pack * p.tok_tile && tok < w.len_q;
  const int reach = live ? reach_of(p, w, tok) : 0;
  const int n_mine = s == 0 ? w.count[0] : w.count[1];
  const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
  const uint32_t tS = tmem + lanes + C::COL_S + (C::S_BUFS == 1 ? 0 : 128 * s), tP = tmem + lanes + C::COL_P + 64 * s;
  const uint32_t tO = tmem + lanes + C::COL_O + DV * s;
  const float c = p.sm_scale * LOG2E;
  const bool idle = RANGES && !__any_sync(0xffffffffu, live);   // no row of this warp exists: its scores are not looked at
  // tiles below this one are seen whole by every row of this tile that exists
  const int whole = reach_of(p, w, row_t0) / TILE_N;

  float m_ref = -INFINITY, m_raw = -INFINITY, l = 0.f;    // l: times the factor on the weights
  bool ok = true;
  auto wait = [&](uint64_t* b, int parity, int code) {
    if (ok && !mbar_wait_fast(bar(b), parity)) {
      gave_up(code);
      ok = false;
    }
  };
#pragma unroll 1
  for (int i = 0; i < n_mine; ++i) {
    wait(&ctrl.s_full[s], i & 1, ERR_S);
    tc_fence_after_sync();
    if (idle) {
      if (lane == 0) mbar_arrive(bar(&ctrl.s_free[C::S_BUFS == 1 ? 0 : s]));
      // the same order as below: P of this tile is reported once P of the one before has been read,
      // or two reports of one warp could fall into one phase
      if (i > 0) wait(&ctrl.o_done[s], (i - 1) & 1, ERR_O);
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(&ctrl.p_full[s]));
      __syncwarp();
      continue;
    }
    uint32_t x[TILE_N];
#pragma unroll
    for (int k = 0; k < 4; ++k) tmem_ld32(tS + 32 * k, x + 32 * k);
    tmem_ld_wait();
    // The scores are in registers: their columns are free for the other row tile's.
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(&ctrl.s_free[C::S_BUFS == 1 ? 0 : s]));
    const int tile = w.first + (twin ? 2 * i + s : i);
    if (tile >= whole) {
      const int see = reach - tile * TILE_N;
#pragma unroll
      for (int k = 0; k < TILE_N; ++k) x[k] = k < see ? x[k] : 0xff800000u;
    }
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int k = 0; k < TILE_N; k += 2)
      mx[(k >> 1) & 3] = max3(mx[(k >> 1) & 3], __uint_as_float(x[k]), __uint_as_float(x[k + 1]));
    const float top = max3(mx[0], mx[1], max3(mx[2], mx[3], -INFINITY));
    m_raw = max3(m_raw, top, -INFINITY);
    const float top2 = top * c;
    const bool raise = top2 > m_ref + RESCALE_THRESHOLD;       // also the first finite one
    float alpha = 1.f;
    if (raise) {
      alpha = ex2_ftz(m_ref - top2);                               // 0 for the first
      m_ref = top2;
      l *= alpha;
    }
    // the product of the tile before has read P, and O is its result
    if (i > 0) {
      wait(&ctrl.o_done[s], (i - 1) & 1, ERR_O);
      tc_fence_after_sync();
    }
    if (i > 0 && __any_sync(0xffffffffu, raise)) {
#pragma unroll 1
      for (int k = 0; k < DV / 16; ++k) {
        uint32_t o[16];
        tmem_ld16(tO + 16 * k, o);
        tmem_ld_wait();
#pragma unroll
        for (int q = 0; q < 16; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * alpha);
        tmem_st16(tO + 16 * k, o);
      }
    }
    const float ref = m_ref == -INFINITY ? 0.f : m_ref;
    if (!(top2 < INFINITY)) l = NAN;                 // a NaN or infinite score: the row shows it
    const float off = BF16 ? -ref : FP16_LIFT - ref;
    const uint64_t c2 = pair(c, c), minus_ref = pair(off, off);
    uint64_t sum[2] = {0, 0};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t pk[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        float a, b;
        unpair(fma_pair(pair(__uint_as_float(x[32 * q + 2 * j]), __uint_as_float(x[32 * q + 2 * j + 1])), c2, minus_ref), a, b);
        a = ex2_ftz(a);
        b = ex2_ftz(b);
        sum[j & 1] = add_pair(sum[j & 1], pair(a, b));
        pk[j] = pack2<BF16>(a, b);
      }
      tmem_st16(tP + 16 * q, pk);
    }
    float s0, s1, s2, s3;
    unpair(sum[0], s0, s1);
    unpair(sum[1], s2, s3);
    l += (s0 + s1) + (s2 + s3);
    tmem_st_wait();
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(&ctrl.p_full[s]));
  }
  grid_launch_dependents();

  // ---- epilogue --------------------------------------------------------------------------
  if (n_mine > 0) wait(&ctrl.o_done[s], (n_mine - 1) & 1, ERR_O);
  tc_fence_after_sync();
  const bool fail = !ok || *reinterpret_cast<volatile int*>(&ctrl.fail) != 0;
  const int64_t t = static_cast<int64_t>(w.q0) + tok;
  float factor = 0.f;
  const int set = RANGES ? 2 * w.split + (twin ? s : 0) : 0;
  if (live) {
    store_stats(p, set, t, h, m_raw, BF16 ? m_ref : m_ref - FP16_LIFT, l, fail, factor);
    float none;
    if (RANGES && !twin) store_stats(p, set + 1, t, h, -INFINITY, -INFINITY, 0.f, false, none);
    if (RANGES && (!twin || s == 0))
      for (int k = w.last_set; k < 2 * p.n_splits; ++k) store_stats(p, k, t, h, -INFINITY, -INFINITY, 0.f, false, none);
  }
  const bool nothing = m_ref == -INFINITY && l == l;
  const bool bad = *reinterpret_cast<volatile int*>(&ctrl.bad) != 0;
  const int64_t acc = ((static_cast<int64_t>(set) * p.t_q + t) * p.h_q + h) * DV;
#pragma unroll 1
  for (int k = 0; k < DV / 32; ++k) {
    uint32_t o[32];
    if (n_mine > 0) {
      tmem_ld32(tO + 32 * k, o);                               // warp-collective
      tmem_ld_wait();
    }
    float f[32];
#pragma unroll
    for (int q = 0; q < 32; ++q) f[q] = nothing ? 0.f : __uint_as_float(o[q]) * factor;
    if (bad && live) {
      // the values that were cleared, for the rows that see them: their weight is positive,
      // so an infinity stays one (and two of both signs, or a NaN, make a NaN)
      const int from = max(w.look, w.first) * TILE_N, to = min(reach, (w.first + (twin ? w.tiles : n_mine)) * TILE_N);
      for (int j = from; j < to; ++j) {
        if (twin && (((j / TILE_N - w.first) & 1) != s)) continue;
        const uint16_t* vr = static_cast<const uint16_t*>(p.v) + (w.k0 + j) * p.stride_v_t + kvh * p.stride_v_h + 32 * k;
#pragma unroll
        for (int q = 0; q < 32; ++q) {
          const uint32_t u = vr[q];
          if (not_finite2<BF16>(u) & 0x8000u) {
            if constexpr (BF16) f[q] += __uint_as_float(u << 16);
            else f[q] += __half2float(__ushort_as_half(static_cast<unsigned short>(u)));
          }
        }
      }
    }
    if (!live || fail) continue;
    if (RANGES) {
#pragma unroll
      for (int q = 0; q < 32; q += 8)
        st_global_32(p.o_accum + acc + 32 * k + q, __float_as_uint(f[q]), __float_as_uint(f[q + 1]),
                     __float_as_uint(f[q + 2]), __float_as_uint(f[q + 3]), __float_as_uint(f[q + 4]),
                     __float_as_uint(f[q + 5]), __float_as_uint(f[q + 6]), __float_as_uint(f[q + 7]));
    } else {
      uint16_t* d = static_cast<uint16_t*>(p.out) + t * p.stride_o_t + h * p.stride_o_h + 32 * k;
      uint32_t o2[16];
#pragma unroll
      for (int q = 0; q < 16; ++q) o2[q] = pack2<BF16>(f[2 * q], f[2 * q + 1]);
      if (p.sectors) {
#pragma unroll
        for (int q = 0; q < 16; q += 8)
          st_global_32(d + 2 * q, o2[q], o2[q + 1], o2[q + 2], o2[q + 3], o2[q + 4], o2[q + 5], o2[q + 6], o2[q + 7]);
      } else {
#pragma unroll
        for (int q = 0; q < 16; q += 4)
          *reinterpret_cast<uint4*>(d + 2 * q) = make_uint4(o2[q], o2[q + 1], o2[q + 2], o2[q + 3]);
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
}

// Joins the partials of the key ranges: one warp per (token, head), in range order.  A lane looks
// at up to four sets' log-sum-exps, so that no load waits for another one; the values of eight
// sets are in flight at a time.
template <int DV, bool BF16>
__global__ void __launch_bounds__(256)
dense_combine_kernel(const __grid_constant__ DenseParams p) {
  constexpr int PER = DV / 32;
  static_assert(2 * DENSE_MAX_SPLITS <= 128, "four sets a lane");
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (item >= static_cast<int64_t>(p.t_q) * p.h_q) return;
  const int64_t t = item / p.h_q;
  const int h = static_cast<int>(item - t * p.h_q);
  if (t < __ldg(p.cu_q) || t >= __ldg(p.cu_q + p.b)) return;   // a row of no sequence stays as it is
  const int sets = 2 * p.n_splits;
  const int64_t rows = static_cast<int64_t>(p.t_q) * p.h_q;
  float e[4], ml = -INFINITY, top = -INFINITY;
  bool failed = false;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int s = 32 * k + lane;
    float2 v = make_float2(-INFINITY, -INFINITY);
    if (s < sets) v = *reinterpret_cast<const float2*>(p.stat_accum + (s * rows + item) * 2);
    e[k] = v.y;
    failed |= v.y != v.y;
    ml = max3(ml, v.x, -INFINITY);
    top = fmaxf(top, v.y);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    ml = max3(ml, __shfl_xor_sync(0xffffffffu, ml, d), -INFINITY);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  }
  if (__any_sync(0xffffffffu, failed)) top = NAN;              // a failed part, or NaN scores, show
  float w[4], sum = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    // a set that holds anything weighs more than nothing, so that values in it that are not finite show;
    // 2^-149 changes no other number
    w[k] = e[k] == -INFINITY ? 0.f : expf(e[k] - top) + 1.4e-45f;
    sum += w[k];
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  float acc[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) acc[k] = 0.f;
  const float* src = p.o_accum + item * DV + lane * PER;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int used = 32 - __clz(__ballot_sync(0xffffffffu, w[k] != 0.f));      // sets up to the last with weight
    for (int s0 = 32 * k; s0 < 32 * k + used; s0 += 8) {
      float v[8][PER], ws[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ws[j] = __shfl_sync(0xffffffffu, w[k], (s0 + j) & 31);
#pragma unroll
        for (int q = 0; q < PER; ++q) v[j][q] = 0.f;
        if (ws[j] != 0.f) {                                    // (the values of a set without weight are not written)
          const float* a = src + (s0 + j) * rows * DV;
          if constexpr (PER == 4) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(a));
            v[j][0] = f.x, v[j][1] = f.y, v[j][2] = f.z, v[j][3] = f.w;
          } else {
            const float2 f = __ldg(reinterpret_cast<const float2*>(a));
            v[j][0] = f.x, v[j][1] = f.y;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int q = 0; q < PER; ++q) acc[q] = fmaf(ws[j], v[j][q], acc[q]);
    }
  }
  const bool none = top == -INFINITY;
  const float lse = none ? -INFINITY : top + logf(sum);
  float f = none ? 0.f : 1.f / sum;
  if (p.sink != nullptr && !none) f *= 1.f / (1.f + expf(p.sink[h] - lse));
  uint32_t* d = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + t * p.stride_o_t + h * p.stride_o_h + lane * PER);
#pragma unroll
  for (int k = 0; k < PER / 2; ++k) d[k] = pack2<BF16>(acc[2 * k] * f, acc[2 * k + 1] * f);
  if (lane == 0) {
    p.max_logits[t * p.stride_ml_t + h] = ml;
    p.lse[t * p.stride_lse_t + h] = none ? INFINITY : lse;
  }
}

template <int DQK, int DV, bool BF16, bool RANGES>
cudaError_t launch_one(const DenseParams& p, cudaStream_t st) {
  constexpr size_t smem = dense_smem_bytes<DQK, DV>();
  cudaError_t e = allow_shared_memory<dense_attn_kernel<DQK, DV, BF16, RANGES>>(smem);
  if (e) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(RANGES ? p.ctas : p.items));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  cfg.numAttrs = add_overlap_attribute(attr);
  if ((e = cudaLaunchKernelEx(&cfg, dense_attn_kernel<DQK, DV, BF16, RANGES>, p))) return e;
  if (!RANGES) return cudaSuccess;
  cfg.gridDim = dim3(static_cast<unsigned>((static_cast<int64_t>(p.t_q) * p.h_q + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, dense_combine_kernel<DV, BF16>, p);
}

template <int DQK, int DV>
cudaError_t launch_dims(const DenseParams& p, bool bf16, cudaStream_t st) {
  if (p.n_splits > 1) return bf16 ? launch_one<DQK, DV, true, true>(p, st) : launch_one<DQK, DV, false, true>(p, st);
  return bf16 ? launch_one<DQK, DV, true, false>(p, st) : launch_one<DQK, DV, false, false>(p, st);
}

// Heads packed into a row tile: the most heads of a group that divide it and fit.
int pack_of(int group) {
  for (int v = group < TILE_M ? group : TILE_M; v > 1; --v)
    if (group % v == 0) return v;
  return 1;
}

// CTAs of a launch with ranges: one for every SM, or twice the uncut ones where those alone are
// more than half of the SMs.
int64_t dense_range_ctas(int64_t ctas, int num_sms) { return 2 * ctas > num_sms ? 2 * ctas : num_sms; }

}  // namespace

int64_t dense_ctas(int t_q, int b, int h_q, int h_kv) {
  const int pack = pack_of(h_q / h_kv);
  return (static_cast<int64_t>(t_q) / (2 * (TILE_M / pack)) + b) * (h_q / pack);
}

cudaError_t launch_dense_prefill(const Dsv4DensePrefillArgs& a, int num_sms, cudaStream_t st) {
  DenseParams p;
  const bool bf16 = a.dtype == DSV4_DTYPE_BF16;
  p.b = a.b; p.t_q = a.t_q; p.t_k = a.t_k; p.h_q = a.h_q; p.h_kv = a.h_kv; p.causal = a.causal;
  p.pack = pack_of(a.h_q / a.h_kv);
  p.tok_tile = TILE_M / p.pack;
  p.chunks = a.h_q / p.pack;
  p.slots = a.t_q / (2 * p.tok_tile) + a.b;
  p.n_splits = a.n_splits;
  p.items = p.slots * p.chunks;
  p.sms = num_sms;
  p.ctas = static_cast<int>(dense_range_ctas(p.items, num_sms));
  p.sm_scale = a.sm_scale;
  p.cu_q = a.cu_seqlens_q; p.cu_k = a.cu_seqlens_k; p.sink = a.attn_sink;
  p.v = a.v; p.stride_v_t = a.stride_v_t; p.stride_v_h = a.stride_v_h;
  p.out = a.out; p.max_logits = a.max_logits; p.lse = a.lse;
  p.stride_o_t = a.stride_o_t; p.stride_o_h = a.stride_o_h;
  p.stride_ml_t = a.stride_ml_t; p.stride_lse_t = a.stride_lse_t;
  p.o_accum = a.o_accum; p.stat_accum = a.stat_accum;
  p.sectors = ((reinterpret_cast<uintptr_t>(a.out) | (a.stride_o_t * 2) | (a.stride_o_h * 2)) & 31) == 0;
  cudaError_t e;
  if ((e = make_map_16bit(&p.mq, bf16, a.q, a.t_q, a.h_q, a.d_qk, a.stride_q_t, a.stride_q_h, p.tok_tile, p.pack))) return e;
  // a batch without any key still needs legal maps: nothing is loaded through them
  const bool keys = a.t_k > 0;
  if ((e = make_map_16bit(&p.mk, bf16, keys ? a.k : a.q, keys ? a.t_k : 1, keys ? a.h_kv : 1, a.d_qk,
                    a.stride_k_t, a.stride_k_h, TILE_N, 1))) return e;
  if ((e = make_map_16bit(&p.mv, bf16, keys ? a.v : a.q, keys ? a.t_k : 1, keys ? a.h_kv : 1, a.d_v,
                    a.stride_v_t, a.stride_v_h, TILE_N, 1))) return e;
  if (a.d_qk == 192) return launch_dims<192, 128>(p, bf16, st);
  if (a.d_qk == 128) return launch_dims<128, 128>(p, bf16, st);
  return launch_dims<64, 64>(p, bf16, st);
}

cudaError_t read_dense_error(int* value, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(value, g_dense_error, sizeof(int));
  if (e) return e;
  if (reset && *value) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_dense_error, &zero, sizeof(int));
  }
  return e;
}

}  // namespace dsv4
