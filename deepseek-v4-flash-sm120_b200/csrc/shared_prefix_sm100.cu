// Attention of many query rows over one prefix: the shared part of a batch's decode.
//
// The rows of all requests and heads (b * s_q * h_q of them) see the same tokens, so the FP8
// rows of the prefix are converted to BF16 once (shared_setup_kernel), and the products run
// over blocks of 128 query rows as a dense attention with d_qk 576 or 512 and V the first 512
// columns of the same rows.
//
// prefix_attn_kernel.  A pair of SMs (cluster of 2, cta_group::2, M = 128) owns 128 query
// rows, 64 each, and walks tiles of 128 tokens:
//   S [128 rows, 128 tokens] = Q K^T      A = Q: each CTA its 64 rows; B = K: each CTA 64 tokens
//   O [128 rows, 512]       += P V        A = P: each CTA its rows;   B = V: each CTA 256 columns
// Why a pair: with one SM 64 rows of O fill half of TMEM, but Q (72 KB) and a tile of 128 rows
// (144 KB) leave no room to load the next one, and an M = 128 product of 64 rows (rows as N)
// reads operands faster than shared memory gives them (two thirds of the tensor rate).  In a
// pair each SM holds half of K's tokens and half of V's columns, and cta_group::2 with M = 128
// runs at the full rate (32 clk for N = 128, 64 for N = 256, measured): 2176 clk a tile.
// The CTA's part of an accumulator with M = 128 is its 64 rows, columns [0, N/2) in TMEM lanes
// 0..63 and [N/2, N) in lanes 64..127; so a softmax thread has 64 of a row's 128 scores, and the
// two threads of a row agree on its reference maximum, which is raised only when a score exceeds
// it by 2^8 (one barrier with an OR per tile otherwise).
//
// Nothing waits for the softmax: scores have two buffers in TMEM, so the tensor core works on
// Q K^T of tile t + 1 and P V of tile t - 1 while the exponentials of tile t are formed.  K is
// recycled in groups of blocks as Q K^T passes them, V in halves of its columns.
//
// The requests' own tokens can be attended in the same pass: the tiles of every request with rows
// in a block follow the prefix's, seen by that request's rows only.  That wastes most of such a
// tile's products, but saves a launch that is as long as its longest request (64 requests of 64
// to 2048 own tokens: 45 us; here 6 % more tiles, and 11 us more of conversion).
//
// Work is cut evenly: the tiles of all row blocks form one line that is divided among the
// clusters; a cluster's share is one or more segments (a range of tiles of one row block), each
// leaving a normalised 32-bit partial and its log-sum-exp.  The segments of a row block are its
// sets 0, 1, ...; the last one marks the sets that are not used with -inf.
//
// Measured (64 requests x 64 heads, a prefix of 32768 of d_qk 576, 64 to 2048 own tokens): 191 us,
// 1.5 PFLOP/s for the prefix alone, tensor pipe 91 % busy at an SM clock of 1.43 GHz (both from one
// profile).  Bound by the tensor cores at that clock; around it conversion 26 us and the join 14 us
// (2 KB a row and set read, 1 KB a row written).
#include "attn_params.cuh"
#include "launch_util.h"
#include "launchers.h"
#include "paging.cuh"
#include "sm100_ptx.cuh"
#include "tensor_map.h"

namespace dsv4 {

__device__ int g_prefix_error = 0;

namespace {

using namespace ptx;

constexpr int ROWS = 64;                        // query rows of a CTA
constexpr int TILE = 128;                       // tokens
constexpr int GROUP = 128, SOFTMAX_THREADS = 2 * GROUP;         // two softmax warpgroups
constexpr int THREADS = SOFTMAX_THREADS + 128;                  // and four warps that issue and load
constexpr int WARP_QK = 8, WARP_PV = 9, WARP_LOAD_K = 10, WARP_LOAD_V = 11;
constexpr int BAR_BOTH = 1, BAR_DECIDED = 2, BAR_GROUP = 4;     // named barriers (2 and 3, 4 and 5)
constexpr int QK_BLOCK = ROWS * 128;            // [64 rows or tokens][64 values]: 8 KB
constexpr int V_BLOCK = TILE * 128;             // [128 tokens][64 columns]: 16 KB
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float RESCALE_THRESHOLD = 8.0f;       // log2 units
constexpr uint32_t TMEM_COLS = 512, COL_O = 0, COL_S = 256;     // O 2 x 128, S 2 x 64 columns
constexpr int MIN_TILES = 2;                    // of a cluster's share (drawn calls of this form: 4 takes 6 % longer, 6 14 %)

enum PrefixErr { ERR_Q = 21, ERR_K = 22, ERR_V = 23, ERR_P = 24, ERR_S = 25, ERR_O = 26, ERR_SLOT = 27, ERR_FREE = 28 };

template <int DQK> struct PCfg {
  static constexpr int NB = DQK / 64;
  static constexpr int GROUPS = NB == 9 ? 3 : 4, PER = NB / GROUPS;      // K blocks handed over together
  static constexpr int Q_BYTES = NB * QK_BLOCK, K_BYTES = NB * QK_BLOCK;
  static constexpr int V_BYTES = 4 * V_BLOCK, P_BYTES = ROWS * TILE * 2;
};

struct PrefixCtrl {
  // of each CTA: a commit of the leader's products arrives
  uint64_t k_empty[4], v_empty[2], s_full[2], o_done[2];
  // of the leader: the TMA loads of both CTAs, or the softmax warps of both, report
  uint64_t q_land, k_land[4], v_land[2], s_free[2], p_full, o_free;
  uint32_t tmem;
  int fail;
  alignas(16) float ref[ROWS];
  float part[4][ROWS];           // by group and half: a tile's maxima; at a segment's end the sums
};

template <int DQK> constexpr size_t prefix_smem_bytes() {
  using C = PCfg<DQK>;
  return 1024 + C::Q_BYTES + C::K_BYTES + C::V_BYTES + C::P_BYTES + sizeof(PrefixCtrl);
}
static_assert(prefix_smem_bytes<576>() <= 232448, "227 KB a CTA");

struct PrefixParams {
  CUtensorMap mq, mk, mv;        // query rows; token rows in boxes of 64 and of 128
  int rows, sets, blocks;        // query rows, partial sets, blocks of 128 rows
  int max_tokens, padded;        // of the prefix: tokens, and rows of the workspace
  int own_max, own_padded;       // of each request's own tokens; 0: attended elsewhere
  int b, s_q, h_q;
  const int32_t *length, *own;   // [1], [b]
  const int32_t* starts;         // [blocks + 2]: where a block's tiles start; the most of a block
  const uint32_t *valid, *unfit; // one bit a row of the workspace: it exists; it is not finite
  float sm_scale;
  float *o_accum, *lse_accum;    // [sets][rows][512], [sets][rows]
};

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The leader's barrier at the same offset as `bar` here.
__device__ __forceinline__ uint32_t of_leader(uint32_t bar) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(bar));
  return a;
}
// Arrive on the leader's barrier.  What the softmax warps report is read by the tensor core
// alone, out of the reporting CTA's own shared memory and TMEM: P (written, then
// fence.proxy.async) or TMEM (tcgen05 fences).  No thread reads another CTA's memory, so the
// arrival releases at CTA scope; releasing and acquiring at cluster scope took 270 to 1300 clk.
__device__ __forceinline__ void arrive_leader(uint32_t bar) {
  const uint32_t a = of_leader(bar);
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(a) : "memory");
}
// A box into this CTA's shared memory, reported to a barrier of either CTA of the pair.
__device__ __forceinline__ void load_pair(uint32_t dst, const void* map, int x, int y, int z, uint32_t cluster_bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void umma2(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(elected) : "memory");
}
// Arrive on the barrier at this offset in both CTAs once the products issued so far are done.
__device__ __forceinline__ void commit2(uint32_t bar, uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t.reg .b16 m;\n\t"
      "mov.b16 m, 3;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}"
      ::"r"(bar), "r"(elected) : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&t);
}

// How many own tokens request r has.
__device__ __forceinline__ int own_tokens(const PrefixParams& p, int r) { return min(max(__ldg(p.own + r), 0), p.own_max); }

// This cluster's share of the line of tiles, segment by segment.  Used by whole warps.
struct Share {
  int blocks, prefix_tiles;
  int per, at, end;              // tiles of a cluster; where it is, where it ends
  int block, first, count, set;  // the current segment: tiles [first, first + count) of a block,
  int shared;                    // of which the first `shared` are the prefix's
  bool last;                     // it ends its row block
  __device__ __forceinline__ Share(const PrefixParams& p, int cluster, int clusters) {
    const int len = __ldg(p.length), line = __ldg(p.starts + p.blocks), most = __ldg(p.starts + p.blocks + 1);
    blocks = p.blocks;
    prefix_tiles = (min(max(len, 0), p.max_tokens) + TILE - 1) / TILE;
    // an even share, but no block in more than p.sets segments: its tiles / per + 1 at most
    per = max(max((line + clusters - 1) / clusters, (most + p.sets - 2) / (p.sets - 1)), MIN_TILES);
    at = static_cast<int>(min(static_cast<int64_t>(cluster) * per, static_cast<int64_t>(line)));
    end = static_cast<int>(min(static_cast<int64_t>(at) + per, static_cast<int64_t>(line)));
  }
  __device__ __forceinline__ bool next(const int32_t* starts) {
    if (at >= end) return false;
    // the last block that starts at or before `at`, 32 candidates at a time
    const int lane = threadIdx.x & 31;
    int lo = 0, n = blocks;
    while (n > 1) {
      const int step = (n + 31) / 32;
      const bool below = lane * step < n && __ldg(starts + lo + lane * step) <= at;
      const int hit = 31 - __clz(__ballot_sync(0xffffffffu, below) | 1u);
      n = min(step, n - hit * step);
      lo += hit * step;
    }
    block = lo;
    const int begin = __ldg(starts + lo), tiles = __ldg(starts + lo + 1) - begin;
    first = at - begin;
    count = min(end - at, tiles - first);
    shared = min(count, max(prefix_tiles - first, 0));
    // segments of this block before this one: shares that begin in it, and the one it begins in
    set = at / per - begin / per;
    last = first + count == tiles;
    at += count;
    return true;
  }
};

// The tiles of own tokens of a block one after the other, from the `skip`-th on: of each request
// with rows in the block.  The roles walk them in loops of their own behind the prefix's, whose
// loops stay as short as they can be: with one loop for both the prefix's tiles took 18 % longer.
struct OwnTile {
  int req, own, len;             // the request, which tile of its tokens, and how many it has
  __device__ __forceinline__ OwnTile(const PrefixParams& p, int block, int skip) {
    req = block * 2 * ROWS / (p.s_q * p.h_q) - 1;
    own = len = 0;
    for (; skip >= 0; --skip) step(p);
  }
  __device__ __forceinline__ void step(const PrefixParams& p) {
    if (++own * TILE < len) return;
    own = 0;
    for (len = 0; len == 0 && req + 1 < p.b;) len = own_tokens(p, ++req);
  }
  // first row of the workspace
  __device__ __forceinline__ int row(const PrefixParams& p) const { return p.padded + req * p.own_padded + own * TILE; }
};

template <int DQK>
__global__ void __launch_bounds__(THREADS, 1)
prefix_attn_kernel(const __grid_constant__ PrefixParams p) {
  using C = PCfg<DQK>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t sQ = base, sK = sQ + C::Q_BYTES, sV = sK + C::K_BYTES, sP = sV + C::V_BYTES;
  PrefixCtrl& ctrl = *reinterpret_cast<PrefixCtrl*>(smem_raw + (base - raw) + C::Q_BYTES + C::K_BYTES + C::V_BYTES + C::P_BYTES);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cta_rank();
  auto bar = [&](uint64_t* x) { return smem_u32(x); };

  if (warp == WARP_QK) {
    if (lane == 0) {
      mbar_init(bar(&ctrl.q_land), 1);
      for (int g = 0; g < 4; ++g) {
        mbar_init(bar(&ctrl.k_land[g]), 1);
        mbar_init(bar(&ctrl.k_empty[g]), 1);
      }
      for (int h = 0; h < 2; ++h) {
        mbar_init(bar(&ctrl.v_land[h]), 1);
        mbar_init(bar(&ctrl.v_empty[h]), 1);
        mbar_init(bar(&ctrl.s_full[h]), 1);
        mbar_init(bar(&ctrl.s_free[h]), 8);      // four softmax warps of each CTA
        mbar_init(bar(&ctrl.o_done[h]), 1);
      }
      mbar_init(bar(&ctrl.p_full), 8);
      mbar_init(bar(&ctrl.o_free), 16);
      ctrl.fail = 0;
      mbar_init_fence();
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&ctrl.tmem)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == WARP_LOAD_K && lane == 0) {
    tma_prefetch_map(&p.mq);
    tma_prefetch_map(&p.mk);
    tma_prefetch_map(&p.mv);
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();                                // the other CTA's barriers and TMEM are there too
  tc_fence_after_sync();
  const uint32_t tmem = ctrl.tmem;
  grid_dependency_wait();
  Share w(p, blockIdx.x >> 1, gridDim.x >> 1);
  // A lane whose bounded wait gives up records it, waits for nothing any more, and issues and reports
  // nothing (its arrivals would stand in for the other CTA's, whose rows would be wrong and not know);
  // but it walks on through the same loops, so that its warp stays together for what the whole warp has
  // to execute (a phase may complete just as the first lanes give up) and every barrier of the CTA
  // is met.
  bool ok = true;
  auto gave_up = [&](int code) {
    atomicExch(&g_prefix_error, code);
    *reinterpret_cast<volatile int*>(&ctrl.fail) = 1;
    ok = false;
  };

  if (warp >= WARP_QK) {
    const uint32_t elected = elect_one();          // the lane that loads or issues
    auto wait = [&](uint64_t* b, int parity, int code) {
      if (ok && !mbar_wait_fast(bar(b), parity)) {
        if (elected) gave_up(code);
        ok = false;
      }
    };                                 // (no lane needs another one until the next segment; a __syncwarp
                                       // took 1 % more)
    if (warp == WARP_LOAD_K) {
      // ======================= Q and K ======================================================
      int n = 0;
      while (__all_sync(0xffffffffu, ok) && w.next(p.starts)) {
        // Q is free once every product of the segment before is done
        for (int g = 0; g < C::GROUPS; ++g) wait(&ctrl.k_empty[g], (n & 1) ^ 1, ERR_SLOT);
        if (ok && elected) {
          if (rank == 0) mbar_expect_tx(bar(&ctrl.q_land), 2 * C::Q_BYTES);
          for (int c = 0; c < C::NB; ++c)
            load_pair(sQ + c * QK_BLOCK, &p.mq, 64 * c, 0, w.block * 2 * ROWS + rank * ROWS, of_leader(bar(&ctrl.q_land)));
        }
        auto load = [&](int tok) {
          tok += rank * ROWS;
          for (int g = 0; g < C::GROUPS; ++g) {
            wait(&ctrl.k_empty[g], (n & 1) ^ 1, ERR_SLOT);
            if (ok && elected) {
              if (rank == 0) mbar_expect_tx(bar(&ctrl.k_land[g]), 2 * C::PER * QK_BLOCK);
              for (int c = g * C::PER; c < (g + 1) * C::PER; ++c)
                load_pair(sK + c * QK_BLOCK, &p.mk, 64 * c, 0, tok, of_leader(bar(&ctrl.k_land[g])));
            }
          }
          ++n;
        };
        int i = 0;
        for (; i < w.shared; ++i) load((w.first + i) * TILE);
        if (i < w.count) {
          OwnTile tile(p, w.block, w.first + i - w.prefix_tiles);
          for (; i < w.count; ++i) {
            load(tile.row(p));
            tile.step(p);
          }
        }
      }
    } else if (warp == WARP_LOAD_V) {
      // ======================= V ============================================================
      int n = 0;
      while (__all_sync(0xffffffffu, ok) && w.next(p.starts)) {
        auto load = [&](int tok) {
          for (int h = 0; h < 2; ++h) {
            wait(&ctrl.v_empty[h], (n & 1) ^ 1, ERR_SLOT);
            if (ok && elected) {
              if (rank == 0) mbar_expect_tx(bar(&ctrl.v_land[h]), 4 * V_BLOCK);
              for (int c = 0; c < 2; ++c)
                load_pair(sV + (2 * h + c) * V_BLOCK, &p.mv, 256 * h + 128 * rank + 64 * c, 0, tok, of_leader(bar(&ctrl.v_land[h])));
            }
          }
          ++n;
        };
        int i = 0;
        for (; i < w.shared; ++i) load((w.first + i) * TILE);
        if (i < w.count) {
          OwnTile tile(p, w.block, w.first + i - w.prefix_tiles);
          for (; i < w.count; ++i) {
            load(tile.row(p));
            tile.step(p);
          }
        }
      }
    } else if (rank != 0) {
      // the leader issues the products of both CTAs
    } else if (warp == WARP_QK) {
      // ======================= scores (leader) ==============================================
      constexpr uint32_t idesc = make_idesc_bf16(128, TILE, 0, 0);
      const uint64_t dQ = make_smem_desc(sQ, 16, 1024, SWZ_128B), dK = make_smem_desc(sK, 16, 1024, SWZ_128B);
      const uint32_t t0 = __shfl_sync(0xffffffffu, tmem, 0) + COL_S;
      int n = 0, seg = 0;
      while (__all_sync(0xffffffffu, ok) && w.next(p.starts)) {
        wait(&ctrl.q_land, seg & 1, ERR_Q);
        ++seg;
        const int count = __shfl_sync(0xffffffffu, w.count, 0);
#pragma unroll 1
        for (int i = 0; i < count; ++i, ++n) {
          wait(&ctrl.s_free[n & 1], ((n >> 1) & 1) ^ 1, ERR_FREE);
          const uint32_t tS = t0 + 64 * (n & 1);
#pragma unroll
          for (int g = 0; g < C::GROUPS; ++g) {
            wait(&ctrl.k_land[g], n & 1, ERR_K);
            tc_fence_after_sync();
            if (!ok) continue;
#pragma unroll
            for (int k = 0; k < 4 * C::PER; ++k) {
              const uint32_t off = ((g * C::PER + (k >> 2)) * QK_BLOCK + (k & 3) * 32) >> 4;
              umma2(tS, dQ + off, dK + off, idesc, (g | k) != 0, elected);
            }
            commit2(bar(&ctrl.k_empty[g]), elected);
          }
          if (ok) commit2(bar(&ctrl.s_full[n & 1]), elected);
        }
      }
    } else {
      // ======================= products with V (leader) =====================================
      constexpr uint32_t idesc = make_idesc_bf16(128, 256, 0, 1);
      const uint64_t dP = make_smem_desc(sP, 16, 1024, SWZ_128B);
      const uint64_t dV = make_smem_desc(sV, V_BLOCK, 1024, SWZ_128B);       // MN-major
      const uint32_t t0 = __shfl_sync(0xffffffffu, tmem, 0) + COL_O;
      int n = 0, seg = 0;
      while (__all_sync(0xffffffffu, ok) && w.next(p.starts)) {
        wait(&ctrl.o_free, (seg & 1) ^ 1, ERR_FREE);     // the segment before has been read out
        ++seg;
        const int count = __shfl_sync(0xffffffffu, w.count, 0);
#pragma unroll 1
        for (int i = 0; i < count; ++i, ++n) {
          wait(&ctrl.p_full, n & 1, ERR_P);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            wait(&ctrl.v_land[h], n & 1, ERR_V);
            tc_fence_after_sync();
            if (!ok) continue;
#pragma unroll
            for (int k = 0; k < TILE / 16; ++k)
              umma2(t0 + 128 * h, dP + (((k >> 2) * QK_BLOCK + (k & 3) * 32) >> 4),
                    dV + ((2 * h * V_BLOCK + k * 2048) >> 4), idesc, (i | k) != 0, elected);
            commit2(bar(&ctrl.v_empty[h]), elected);
          }
          if (ok) commit2(bar(&ctrl.o_done[n & 1]), elected);
        }
      }
    }
  } else {
    // ======================= softmax =======================================================
    // The two warpgroups take the tiles in turn (tile n: group n & 1), so that one's waits and
    // stores hide behind the other's arithmetic.  Thread l of a group: row l & 63, tokens
    // [64 * (l >> 6), +64) of the tile.  The rows' reference maxima are common (they scale O):
    // a group decides about raising them once the other one has decided for the tile before.
    const int group = tid >> 7, r = tid & 63, half = (tid >> 6) & 1;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const float c = p.sm_scale * LOG2E;
    const uint32_t prow = sP + half * QK_BLOCK + r * 128;
    auto wait = [&](uint64_t* b, int parity, int code) {
      if (ok && !mbar_wait_fast(bar(b), parity)) gave_up(code);
    };
    const int64_t total_tiles = w.end - w.at;
    int n = 0;
    while (w.next(p.starts)) {
      if (tid < ROWS) ctrl.ref[tid] = -INFINITY;
      bar_sync(BAR_BOTH, SOFTMAX_THREADS);
      float m_ref = -INFINITY, l = 0.f;            // l is relative to m_ref
      const int mine = (n & 1) == group ? 0 : 1;   // this group's first tile of the segment
      const int n0 = n;                            // tiles of the segments before
      const int row = w.block * 2 * ROWS + rank * ROWS + r;
      // Tile i of the segment; of this thread's 64 tokens its row sees those whose bits are set.
      auto attend = [&](int i, uint2 seen) {
        n = n0 + i;
        wait(&ctrl.s_full[group], (n >> 1) & 1, ERR_S);
        tc_fence_after_sync();
        uint32_t x[64];
        tmem_ld32(tmem + lanes + COL_S + 64 * group, x);
        tmem_ld32(tmem + lanes + COL_S + 64 * group + 32, x + 32);
        tmem_ld_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0 && ok) arrive_leader(bar(&ctrl.s_free[group]));
        if ((seen.x & seen.y) != 0xffffffffu) {
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            if (!((seen.x >> k) & 1u)) x[k] = 0xff800000u;
            if (!((seen.y >> k) & 1u)) x[32 + k] = 0xff800000u;
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < 64; ++k) mx[k & 3] = fmaxf(mx[k & 3], __uint_as_float(x[k]));
        const float top2 = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;

        if (n > 0) bar_sync(BAR_DECIDED + (group ^ 1), SOFTMAX_THREADS);
        float ref = ctrl.ref[r];
        if (bar_red_or(BAR_GROUP + group, GROUP, top2 > ref + RESCALE_THRESHOLD)) {
          // some row's reference is raised (always in a segment's first tile)
          ctrl.part[2 * group + half][r] = top2;
          bar_sync(BAR_GROUP + group, GROUP);
          const float both = fmaxf(top2, ctrl.part[2 * group + (half ^ 1)][r]);
          float alpha = 1.f;
          if (both > ref + RESCALE_THRESHOLD) {
            alpha = ex2_ftz(ref - both);               // 0 for the first
            ref = both;
          }
          bar_sync(BAR_GROUP + group, GROUP);      // both threads of a row have read the old one
          if (half == 0) ctrl.ref[r] = ref;
          if (i > 0) {
            wait(&ctrl.o_done[group ^ 1], ((n - 1) >> 1) & 1, ERR_O);
            tc_fence_after_sync();
            if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
              for (int k = 0; k < 16; ++k) {
                uint32_t o[16];
                tmem_ld16(tmem + lanes + COL_O + 16 * k, o);
                tmem_ld_wait();
#pragma unroll
                for (int q = 0; q < 16; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * alpha);
                tmem_st16(tmem + lanes + COL_O + 16 * k, o);
              }
              tmem_st_wait();
            }
          }
        }
        if (n + 1 < total_tiles) bar_arrive(BAR_DECIDED + group, SOFTMAX_THREADS);
        if (ref != m_ref) {                        // raised here or by the other group
          l *= ex2_ftz(m_ref - ref);
          m_ref = ref;
        }
        const float sub = ref == -INFINITY ? 0.f : ref;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t pk[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const float a = ex2_ftz(fmaf(__uint_as_float(x[2 * k]), c, -sub));
          const float b = ex2_ftz(fmaf(__uint_as_float(x[2 * k + 1]), c, -sub));
          sum[(2 * k) & 3] += a;
          sum[(2 * k + 1) & 3] += b;
          pk[k] = pack_bf16x2(a, b);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        // P V of the tile before has read P
        if (n > 0) wait(&ctrl.o_done[group ^ 1], ((n - 1) >> 1) & 1, ERR_O);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(prow + ((k ^ (r & 7)) << 4)), "r"(pk[4 * k]),
                       "r"(pk[4 * k + 1]), "r"(pk[4 * k + 2]), "r"(pk[4 * k + 3]) : "memory");
        fence_async_smem();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0 && ok) arrive_leader(bar(&ctrl.p_full));
      };
      // bits are fetched a tile ahead
      const uint2* bits = reinterpret_cast<const uint2*>(p.valid) + w.first * 2 + half;
      int i = mine;
      uint2 ahead = make_uint2(0u, 0u);
      if (i < w.shared) ahead = __ldg(bits + 2 * i);
#pragma unroll 1
      for (; i < w.shared; i += 2) {
        const uint2 seen = ahead;
        if (i + 2 < w.shared) ahead = __ldg(bits + 2 * (i + 2));
        attend(i, seen);
      }
      if (i < w.count) {
        const int rows_of_req = p.s_q * p.h_q, my_req = row / rows_of_req, unseen = p.s_q - 1 - row % rows_of_req / p.h_q;
        OwnTile tile(p, w.block, w.first + i - w.prefix_tiles);
        auto own_bits = [&]() {
          const int64_t at = tile.row(p) >> 5;
          uint2 v = __ldg(reinterpret_cast<const uint2*>(p.valid + at) + half);
          // of this row's request, up to its own place
          const int sees = tile.req == my_req ? tile.len - unseen - tile.own * TILE - 64 * half : 0;
          if (sees < 64) v.y &= sees <= 32 ? 0u : (1u << (sees - 32)) - 1u;
          if (sees < 32) v.x &= sees <= 0 ? 0u : (1u << sees) - 1u;
          // the setup has zeroed what is not finite, for the rows that do not see it
          const uint2 unfit = __ldg(reinterpret_cast<const uint2*>(p.unfit + at) + half);
          if (((unfit.x & v.x) | (unfit.y & v.y)) != 0u) l = NAN;
          return v;
        };
        ahead = own_bits();
#pragma unroll 1
        for (; i < w.count; i += 2) {
          const uint2 seen = ahead;
          if (i + 2 < w.count) {
            tile.step(p);
            tile.step(p);
            ahead = own_bits();
          }
          attend(i, seen);
        }
      }
      n = n0 + w.count;
      // ---- the segment's partial ------------------------------------------------------------
      bar_sync(BAR_BOTH, SOFTMAX_THREADS);         // every decision has been made
      const float ref = ctrl.ref[r];
      if (ref != m_ref) l *= ex2_ftz(m_ref - ref);
      ctrl.part[2 * group + half][r] = l;
      bar_sync(BAR_BOTH, SOFTMAX_THREADS);
      const float total = (ctrl.part[0][r] + ctrl.part[1][r]) + (ctrl.part[2][r] + ctrl.part[3][r]);
      wait(&ctrl.o_done[(n - 1) & 1], ((n - 1) >> 1) & 1, ERR_O);
      tc_fence_after_sync();
      const bool fail = *reinterpret_cast<volatile int*>(&ctrl.fail) != 0;
      const bool none = total == 0.f;
      const float f = none ? 0.f : 1.f / total;
      if (group == 0 && half == 0 && row < p.rows) {
        // a row that failed, or is NaN, has to come out NaN whatever else is joined with it: +inf does
        // so, being the maximum of the sets, where a NaN could be passed over
        const float lse = logf(total) + ref * LN2;
        p.lse_accum[static_cast<int64_t>(w.set) * p.rows + row] = fail || lse != lse ? INFINITY : none ? -INFINITY : lse;
        if (w.last)
          for (int s = w.set + 1; s < p.sets; ++s) p.lse_accum[static_cast<int64_t>(s) * p.rows + row] = -INFINITY;
      }
      // Each group writes the 256 columns of one product.  Four lanes exchange the blocks of 8
      // columns of their rows first, so that they write 128 bytes of each row in turn (32 bytes at
      // 32 places took 8200 clk a segment; 16 requests 80 us, with this 77).
      const int j = lane & 3;
      float* dst = p.o_accum + (static_cast<int64_t>(w.set) * p.rows + row - j) * D_V + group * 256 + half * 128 + 8 * j;
#pragma unroll 1
      for (int k = 0; k < 4; ++k) {
        uint32_t o[32];
        tmem_ld32(tmem + lanes + COL_O + 128 * group + 32 * k, o);             // warp-collective
        tmem_ld_wait();
        if (k == 3) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0 && ok) arrive_leader(bar(&ctrl.o_free));
        }
#pragma unroll
        for (int q = 0; q < 32; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * f);
        // block i of lane j <-> block j of lane i
#pragma unroll
        for (int bit = 1; bit < 4; bit <<= 1) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (i & bit) continue;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const bool up = (j & bit) != 0;
              const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? o[8 * i + q] : o[8 * (i | bit) + q], bit);
              if (up) o[8 * i + q] = got;
              else o[8 * (i | bit) + q] = got;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (row - j + i < p.rows && !fail)
            st_global_32(dst + i * D_V + 32 * k, o[8 * i], o[8 * i + 1], o[8 * i + 2], o[8 * i + 3], o[8 * i + 4],
                         o[8 * i + 5], o[8 * i + 6], o[8 * i + 7]);
      }
    }
    // blocks without any tile: nobody else marks the sets of their rows
    for (int k = blockIdx.x >> 1; k < p.blocks; k += gridDim.x >> 1) {
      if (__ldg(p.starts + k) != __ldg(p.starts + k + 1)) continue;
      const int row = k * 2 * ROWS + rank * ROWS + tid;
      if (tid < ROWS && row < p.rows)
        for (int i = 0; i < p.sets; ++i) p.lse_accum[static_cast<int64_t>(i) * p.rows + row] = -INFINITY;
    }
  }
  grid_launch_dependents();
  // Neither CTA may leave, or free its TMEM, while the other still reports to it.
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();
  tc_fence_after_sync();
  if (warp == WARP_QK)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
}

// Is one of two BF16 numbers an infinity or NaN?
__device__ __forceinline__ bool not_finite(uint32_t two) {
  return (two & 0x7f80u) == 0x7f80u || (two & 0x7f800000u) == 0x7f800000u;
}

// starts[k]: tiles of the row blocks before block k (the prefix's, and of the own tokens of every
// request with rows in the block); then their sum, and the most tiles of a block.  One CTA of 256.
__device__ __forceinline__ void block_starts(const Dsv4SharedPrefixArgs& a, const SharedSetup& out, int prefix) {
  __shared__ int part[8], top[8];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rows_of_req = a.s_q * a.h_q, rows = a.b * rows_of_req, blocks = (rows + 2 * ROWS - 1) / (2 * ROWS);
  const int prefix_tiles = (prefix + TILE - 1) / TILE;
  int carry = 0, most = 0;
  for (int k0 = 0; k0 < blocks; k0 += 256) {
    const int k = k0 + tid;
    int n = 0;
    if (k < blocks) {
      n = prefix_tiles;
      if (out.own_padded > 0)
        for (int r = k * 2 * ROWS / rows_of_req; r <= (min((k + 1) * 2 * ROWS, rows) - 1) / rows_of_req; ++r)
          n += (min(max(a.suffix_length[r], 0), a.max_pages * a.page_block_size) + TILE - 1) / TILE;
    }
    most = max(most, n);
    int sum = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    if (lane == 31) part[warp] = sum;
    __syncthreads();
    int before = carry, all = carry;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < warp) before += part[i];
      all += part[i];
    }
    if (k < blocks) out.starts[k] = before + sum - n;
    carry = all;
    __syncthreads();
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
  if (lane == 0) top[warp] = most;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < 8; ++i) most = max(most, top[i]);
    out.starts[blocks] = carry;
    out.starts[blocks + 1] = most;
  }
}

// One launch for what the attention kernels read besides the cache.  CTAs [0, row_ctas): FP8 rows
// of the prefix, and of every request's own tokens, -> BF16 rows [tokens, d_qk], and a bit per
// token that says whether it exists; rows that do not are zero.  Whole tiles of 128 tokens are
// written.  Bound by memory: 644 (584) B in and 1152 (1024) B out per token; a warp has four
// tokens in flight (32768 tokens and 64 x 1000 own ones: 26 us, writes that stay in L2 among them).
// One CTA: where the row blocks' tiles start.  CTAs [row_ctas, +list_ctas): token indices of the
// prefix.  The others: one query token's list each, of its own tokens or of
// the prefix and those.  List entries behind a length are not written: nothing reads them.
template <int FMT>
__global__ void __launch_bounds__(256)
shared_setup_kernel(const Dsv4SharedPrefixArgs a, const SharedSetup out, const FastDiv page, int row_ctas, int list_ctas) {
  using T = KvTraits<FMT>;
  grid_dependency_wait();
  grid_launch_dependents();        // the next kernel sets itself up meanwhile, and waits for this one
  const int prefix = a.prefix_pages > 0 ? min(max(*a.prefix_length, 0), a.prefix_pages * a.page_block_size) : 0;
  const int n_tok = a.num_blocks * a.page_block_size;
  auto entry = [&](const int32_t* table, int pages, int pos) {
    const int s = slot_of(table, pages, page, pos);
    return s < n_tok ? s : -1;
  };
  if (static_cast<int>(blockIdx.x) >= row_ctas) {
    int x = blockIdx.x - row_ctas;
    if (out.starts != nullptr) {
      if (x == 0) {
        block_starts(a, out, prefix);
        return;
      }
      --x;
    }
    if (x < list_ctas) {
      for (int j = x * 256 + threadIdx.x; j < prefix; j += list_ctas * 256)
        out.prefix_list[j] = entry(a.prefix_table, a.prefix_pages, j);
      return;
    }
    x -= list_ctas;
    const int r = x / a.s_q, s = x % a.s_q;
    const int width = a.max_pages * a.page_block_size;
    const int own = a.max_pages > 0 ? min(max(a.suffix_length[r], 0), width) : 0;
    const int sees = own - (a.s_q - 1 - s);
    const int32_t* table = a.block_table + r * a.stride_table;
    if (out.joined != nullptr) {
      int32_t* list = out.joined + static_cast<int64_t>(x) * (a.prefix_pages * a.page_block_size + width);
      for (int j = threadIdx.x; j < prefix; j += 256) list[j] = entry(a.prefix_table, a.prefix_pages, j);
      for (int j = threadIdx.x; j < own; j += 256) list[prefix + j] = j < sees ? entry(table, a.max_pages, j) : -1;
      if (s == 0 && threadIdx.x == 0) out.lens[r] = prefix + own;
    } else {
      int32_t* list = out.suffix_lists + static_cast<int64_t>(x) * width;
      for (int j = threadIdx.x; j < own; j += 256) list[j] = j < sees ? entry(table, a.max_pages, j) : -1;
    }
    return;
  }

  // 32 rows of the workspace: of the prefix, or behind those of a request's own tokens
  const int row0 = blockIdx.x * 32;
  int tok0 = row0, len = prefix;
  const int32_t* table = a.prefix_table;
  const bool own = row0 >= out.padded;
  if (own) {
    const int r = (row0 - out.padded) / out.own_padded;
    tok0 = (row0 - out.padded) - r * out.own_padded;
    len = min(max(a.suffix_length[r], 0), a.max_pages * a.page_block_size);
    table = a.block_table + r * a.stride_table;
  }
  if (tok0 >= (len + TILE - 1) / TILE * TILE) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // every warp knows where the CTA's 32 tokens live: lane i looks up token i
  const int tok = tok0 + lane;
  const int col = static_cast<int>(div_by(static_cast<uint32_t>(tok), page));
  int id = -1;
  if (tok < len) id = __ldg(table + col);
  const bool live = id >= 0 && id < a.num_blocks;
  const uint32_t word = __ballot_sync(0xffffffffu, live);
  if (threadIdx.x == 0) out.valid[blockIdx.x] = word;
  const int off = tok - col * a.page_block_size;

  // A tile of own tokens is multiplied with the rows of other requests too, with weights of zero;
  // so that zero times it is zero, a row whose values are not finite is written as zeros and noted
  // (the values are the first 512 numbers: of MODEL1 the rotary part too).
  __shared__ uint32_t noted[8];
  uint32_t unfit = 0;

  const uint8_t* kv = static_cast<const uint8_t*>(a.kv);
  uint4 latent[4], rope[4];
  uint32_t scale[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int i = warp * 4 + k;
    const int pg = __shfl_sync(0xffffffffu, id, i), at = __shfl_sync(0xffffffffu, off, i);
    latent[k] = rope[k] = make_uint4(0, 0, 0, 0);
    scale[k] = 127;
    if ((word >> i) & 1u) {
      const uint8_t* base = kv + static_cast<int64_t>(pg) * a.stride_kv_block;
      const uint8_t* row = base + static_cast<int64_t>(at) * T::ROW_BYTES;
      if (lane < T::D_NOPE / 16) {
        latent[k] = __ldg(reinterpret_cast<const uint4*>(row) + lane);
        scale[k] = __ldg(base + static_cast<int64_t>(a.page_block_size) * T::ROW_BYTES + at * T::SLOTS + lane * 16 / T::TILE);
      }
      if (lane < 8) rope[k] = __ldg(reinterpret_cast<const uint4*>(row + T::D_NOPE) + lane);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out.rows) + static_cast<int64_t>(row0 + warp * 4 + k) * T::D_QK);
    uint32_t o[8] = {};
    if (lane < T::D_NOPE / 16) {
      const ScalePair c = scale_pair(scale[k]);
      const bool two = scale[k] > MAX_ONE_MULTIPLY_SCALE;
      dequant4(latent[k].x, c, two, o[0], o[1]);
      dequant4(latent[k].y, c, two, o[2], o[3]);
      dequant4(latent[k].z, c, two, o[4], o[5]);
      dequant4(latent[k].w, c, two, o[6], o[7]);
    }
    if (own) {
      bool wild = false;
#pragma unroll
      for (int q = 0; q < 8; ++q) wild |= not_finite(o[q]);
      if (T::D_NOPE < D_V) wild |= not_finite(rope[k].x) || not_finite(rope[k].y) || not_finite(rope[k].z) || not_finite(rope[k].w);
      if (__any_sync(0xffffffffu, wild)) {
        unfit |= 1u << (warp * 4 + k);
#pragma unroll
        for (int q = 0; q < 8; ++q) o[q] = 0;
        rope[k] = make_uint4(0, 0, 0, 0);
      }
    }
    if (lane < T::D_NOPE / 16) {
      dst[2 * lane] = make_uint4(o[0], o[1], o[2], o[3]);
      dst[2 * lane + 1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
    if (lane < 8) dst[T::D_NOPE / 8 + lane] = rope[k];
  }
  if (!own) return;
  if (lane == 0) noted[warp] = unfit;
  __syncthreads();
  if (threadIdx.x < 32) {
    const uint32_t all = __reduce_or_sync(0xffffffffu, lane < 8 ? noted[lane] : 0u);
    if (lane == 0) out.unfit[blockIdx.x] = all;
  }
}

// Joins the partial sets of many rows: one warp per (row, head), which has the whole 2 KB of four
// sets in flight; sets in order, so that the result does not depend on timing.  NaN in any of a
// row's log-sum-exps makes the row NaN.  Bound by the latency of its rounds of loads: 4096 rows of
// three or four sets 12.5 us (27 MB), 1024 rows of ten 9.
__global__ void __launch_bounds__(256)
join_sets_kernel(const Dsv4CombineArgs a) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(a.n_rows) * a.h_q;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (item >= rows) return;
  const int row = static_cast<int>(item / a.h_q), h = static_cast<int>(item - static_cast<int64_t>(row) * a.h_q);
  auto lse_of = [&](int set) { return set < a.n_splits ? a.lse_accum[set * rows + item] : -INFINITY; };
  float m = -INFINITY;
  bool failed = false;
  for (int s = lane; s < a.n_splits; s += 32) {
    const float e = lse_of(s);
    failed |= e != e;
    m = fmaxf(m, e);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (__any_sync(0xffffffffu, failed)) m = NAN;
  auto weight_of = [&](int set) {
    const float e = lse_of(set);
    return e == -INFINITY ? 0.f : expf(e - m);
  };
  float l = 0.f;
  for (int s = lane; s < a.n_splits; s += 32) l += weight_of(s);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  const bool has_sink = a.attn_sink != nullptr;
  float lse_v, ml_v;
  const float f = finalize_row(MODE_DECODE, m, l, has_sink, has_sink ? a.attn_sink[h] : 0.f, lse_v, ml_v);
  float acc[16];
#pragma unroll
  for (int q = 0; q < 16; ++q) acc[q] = 0.f;
  // lane: columns 8 * lane .. +8 of each half of the row
  const float4* src = reinterpret_cast<const float4*>(a.o_accum + item * D_V) + 2 * lane;
  float w = 0.f;
  for (int s0 = 0; s0 < a.n_splits; s0 += 4) {
    if ((s0 & 31) == 0) w = weight_of(s0 + lane);
    float4 v[4][4];
    float ws[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      ws[j] = __shfl_sync(0xffffffffu, w, (s0 + j) & 31);       // (0 behind the last set)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        v[j][q] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (ws[j] != 0.f)                        // (a set without weight may hold anything)
          v[j][q] = __ldg(src + (s0 + j) * rows * (D_V / 4) + (q >> 1) * 64 + (q & 1));
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        acc[4 * q] = fmaf(ws[j], v[j][q].x, acc[4 * q]);
        acc[4 * q + 1] = fmaf(ws[j], v[j][q].y, acc[4 * q + 1]);
        acc[4 * q + 2] = fmaf(ws[j], v[j][q].z, acc[4 * q + 2]);
        acc[4 * q + 3] = fmaf(ws[j], v[j][q].w, acc[4 * q + 3]);
      }
  }
  const int bi = row / a.s_q, si = row % a.s_q;
  if (lane == 0) a.lse[bi * a.stride_lse_b + si * a.stride_lse_s + h * a.stride_lse_h] = lse_v;
  __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + bi * a.stride_o_b + si * a.stride_o_s + h * a.stride_o_h;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t o[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = pack_bf16x2(acc[8 * half + 2 * q] * f, acc[8 * half + 2 * q + 1] * f);
    *reinterpret_cast<uint4*>(dst + half * 256 + 8 * lane) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

template <int DQK>
cudaError_t launch_attn(const PrefixParams& p, int clusters, cudaStream_t st) {
  constexpr size_t smem = prefix_smem_bytes<DQK>();
  cudaError_t e = allow_shared_memory<prefix_attn_kernel<DQK>>(smem);
  if (e) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * clusters);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  cfg.numAttrs = add_overlap_attribute(attr);
  attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
  attr[cfg.numAttrs].val.clusterDim.x = 2;
  attr[cfg.numAttrs].val.clusterDim.y = 1;
  attr[cfg.numAttrs].val.clusterDim.z = 1;
  ++cfg.numAttrs;
  return cudaLaunchKernelEx(&cfg, prefix_attn_kernel<DQK>, p);
}

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

}  // namespace

// Enough for even shares of even blocks (a share is at least line / clusters long, so at most
// clusters / blocks of them lie in a row block, and two reach into it), and one more for uneven ones.
int prefix_attn_sets(int64_t rows, int num_sms) {
  const int64_t blocks = (rows + 2 * ROWS - 1) / (2 * ROWS), clusters = num_sms / 2;
  return static_cast<int>((clusters + blocks - 1) / blocks + 2);
}

namespace {
struct Places {
  int64_t padded, own_padded, rows, blocks, unfit, starts, values, bytes;
};
Places places(const Dsv4SharedPrefixArgs& a, bool own) {
  Places x;
  x.padded = round_up(static_cast<int64_t>(a.prefix_pages) * a.page_block_size, TILE);
  x.own_padded = own ? round_up(static_cast<int64_t>(a.max_pages) * a.page_block_size, TILE) : 0;
  x.rows = x.padded + x.own_padded * a.b;
  x.blocks = (static_cast<int64_t>(a.b) * a.s_q * a.h_q + 2 * ROWS - 1) / (2 * ROWS);
  x.unfit = round_up(x.rows / 8, 256);                         // two sets of bits first
  x.starts = 2 * x.unfit;
  x.values = x.starts + round_up((x.blocks + 2) * 4, 256);
  x.bytes = x.values + x.rows * a.d_qk * 2;
  return x;
}
}  // namespace

int64_t prefix_attn_workspace(const Dsv4SharedPrefixArgs& a, bool own) { return places(a, own).bytes; }

bool prefix_attn_fits(const Dsv4SharedPrefixArgs& a, bool own) {
  const Places x = places(a, own);
  const int64_t most = 0x7fffffff - 65536;
  // rows, and the tiles of all blocks (a request's are counted in each block that it has rows in),
  // as 32-bit numbers with room for what is added to them
  return x.rows <= most && x.blocks * (x.padded / TILE) + (x.blocks + a.b) * (x.own_padded / TILE) <= most;
}

void prefix_attn_place(const Dsv4SharedPrefixArgs& a, bool own, SharedSetup& out) {
  const Places x = places(a, own);
  uint8_t* base = static_cast<uint8_t*>(a.workspace);
  out.valid = reinterpret_cast<uint32_t*>(base);
  out.unfit = reinterpret_cast<uint32_t*>(base + x.unfit);
  out.starts = reinterpret_cast<int32_t*>(base + x.starts);
  out.rows = base + x.values;
  out.padded = static_cast<int>(x.padded);
  out.own_padded = static_cast<int>(x.own_padded);
}

cudaError_t launch_shared_setup(const Dsv4SharedPrefixArgs& a, const SharedSetup& out, cudaStream_t st) {
  const int64_t tokens = static_cast<int64_t>(a.prefix_pages) * a.page_block_size;
  const int row_ctas = out.rows != nullptr ? static_cast<int>((out.padded + static_cast<int64_t>(out.own_padded) * a.b) / 32) : 0;
  const int list_ctas = out.prefix_list == nullptr ? 0 : static_cast<int>(tokens < 64 * 1024 ? (tokens + 1023) / 1024 : 64);
  const int lists = out.suffix_lists != nullptr || out.joined != nullptr ? a.b * a.s_q : 0;
  const int starts = out.starts != nullptr ? 1 : 0;
  if (row_ctas + list_ctas + lists + starts == 0) return cudaSuccess;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(row_ctas) + starts + list_ctas + lists);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  cfg.numAttrs = add_overlap_attribute(attr);
  const FastDiv page = fast_div(static_cast<uint32_t>(a.page_block_size));
  return a.kv_format == DSV4_KV_V32
             ? cudaLaunchKernelEx(&cfg, shared_setup_kernel<DSV4_KV_V32>, a, out, page, row_ctas, list_ctas)
             : cudaLaunchKernelEx(&cfg, shared_setup_kernel<DSV4_KV_MODEL1>, a, out, page, row_ctas, list_ctas);
}

cudaError_t launch_join_sets(const Dsv4CombineArgs& a, cudaStream_t st) {
  // Many sets are those of few rows: the combine kernel has a CTA for each row (256 rows of 39 sets:
  // the whole call 52 us with it, 63 with a warp per row).
  if (a.n_splits > 32) return launch_combine(a, st);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((static_cast<int64_t>(a.n_rows) * a.h_q + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  cfg.numAttrs = add_overlap_attribute(attr);
  return cudaLaunchKernelEx(&cfg, join_sets_kernel, a);
}

cudaError_t launch_prefix_attn(const Dsv4SharedPrefixArgs& a, const SharedSetup& setup, int sets, int num_sms, cudaStream_t st) {
  cudaError_t e;
  PrefixParams p;
  p.rows = a.b * a.s_q * a.h_q;
  p.blocks = (p.rows + 2 * ROWS - 1) / (2 * ROWS);
  p.sets = sets;
  p.max_tokens = a.prefix_pages * a.page_block_size;
  p.padded = setup.padded;
  p.own_padded = setup.own_padded;
  p.own_max = setup.own_padded > 0 ? a.max_pages * a.page_block_size : 0;
  p.b = a.b;
  p.s_q = a.s_q;
  p.h_q = a.h_q;
  p.length = a.prefix_length;
  p.own = a.suffix_length;
  p.starts = setup.starts;
  p.valid = setup.valid;
  p.unfit = setup.unfit;
  p.sm_scale = a.sm_scale;
  p.o_accum = a.o_accum;
  p.lse_accum = a.lse_accum;
  const int tokens = setup.padded + setup.own_padded * a.b;
  if ((e = make_map_16bit(&p.mq, true, a.q, p.rows, 1, a.d_qk, a.d_qk, a.d_qk, ROWS, 1))) return e;
  if ((e = make_map_16bit(&p.mk, true, setup.rows, tokens, 1, a.d_qk, a.d_qk, a.d_qk, ROWS, 1))) return e;
  if ((e = make_map_16bit(&p.mv, true, setup.rows, tokens, 1, a.d_qk, a.d_qk, a.d_qk, TILE, 1))) return e;
  return a.d_qk == 576 ? launch_attn<576>(p, num_sms / 2, st) : launch_attn<512>(p, num_sms / 2, st);
}

cudaError_t read_prefix_error(int* value, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(value, g_prefix_error, sizeof(int));
  if (e) return e;
  if (reset && *value) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_prefix_error, &zero, sizeof(int));
  }
  return e;
}

}  // namespace dsv4
