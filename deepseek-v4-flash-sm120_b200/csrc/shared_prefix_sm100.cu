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
// Work is cut evenly: row blocks x tiles form one line that is divided among the clusters; a
// cluster's share is one or more segments (a range of tiles of one row block), each leaving a
// normalised 32-bit partial and its log-sum-exp.  The segments of a row block are its sets
// 0, 1, ...; the last one marks the sets that are not used with -inf.
#include <mutex>

#include "attn_params.cuh"
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
constexpr int MIN_TILES = 4;                    // of a cluster's share

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
  int rows, sets, max_tokens;
  const int32_t* length;         // [1]
  const uint32_t* valid;         // one bit a token
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
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&t);
}

// This cluster's share of the line of row blocks x tiles, segment by segment.
struct Share {
  int tiles;                     // of a row block
  int64_t per, at, end;          // tiles of a cluster; where it is, where it ends
  int block, first, count, set;  // the current segment
  bool last;                     // it ends its row block
  __device__ __forceinline__ Share(const PrefixParams& p, int cluster, int clusters) {
    const int len = min(max(*p.length, 0), p.max_tokens);
    tiles = (len + TILE - 1) / TILE;
    const int64_t line = static_cast<int64_t>(tiles) * ((p.rows + 2 * ROWS - 1) / (2 * ROWS));
    per = max((line + clusters - 1) / clusters, static_cast<int64_t>(MIN_TILES));
    at = min(cluster * per, line);
    end = min(at + per, line);
  }
  __device__ __forceinline__ bool next() {
    if (at >= end) return false;
    block = static_cast<int>(at / tiles);
    first = static_cast<int>(at - static_cast<int64_t>(block) * tiles);
    count = static_cast<int>(min(end - at, static_cast<int64_t>(tiles - first)));
    // segments of this block before this one: shares that begin in it, and the one it begins in
    const int64_t begin = static_cast<int64_t>(block) * tiles;
    set = static_cast<int>(at / per - begin / per);
    last = first + count == tiles;
    at += count;
    return true;
  }
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
  grid_dependency_wait();
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();                                // the other CTA's barriers and TMEM are there too
  tc_fence_after_sync();
  const uint32_t tmem = ctrl.tmem;
  Share w(p, blockIdx.x >> 1, gridDim.x >> 1);
  // A role whose bounded wait gives up records it and waits for nothing any more; what it does
  // from then on is of no use, but every barrier of the CTA is still walked.
  bool ok = true;
  auto gave_up = [&](int code) {
    atomicExch(&g_prefix_error, code);
    *reinterpret_cast<volatile int*>(&ctrl.fail) = 1;
    ok = false;
  };

  if (warp >= WARP_QK) {
    auto wait = [&](uint64_t* b, int parity, int code) {
      if (ok && !mbar_wait_fast(bar(b), parity)) {
        if (lane == 0) gave_up(code);
        ok = false;
      }
      __syncwarp();
    };
    if (warp == WARP_LOAD_K) {
      // ======================= Q and K ======================================================
      const uint32_t elected = elect_one();
      int n = 0;
      while (ok && w.next()) {
        for (int i = 0; i < w.count && ok; ++i, ++n) {
          if (i == 0) {
            // Q is free once every product of the segment before is done
            for (int g = 0; g < C::GROUPS; ++g) wait(&ctrl.k_empty[g], (n & 1) ^ 1, ERR_SLOT);
            if (!ok) break;
            if (elected) {
              if (rank == 0) mbar_expect_tx(bar(&ctrl.q_land), 2 * C::Q_BYTES);
              for (int c = 0; c < C::NB; ++c)
                load_pair(sQ + c * QK_BLOCK, &p.mq, 64 * c, 0, w.block * 2 * ROWS + rank * ROWS, of_leader(bar(&ctrl.q_land)));
            }
          }
          const int tok = (w.first + i) * TILE + rank * ROWS;
          for (int g = 0; g < C::GROUPS; ++g) {
            wait(&ctrl.k_empty[g], (n & 1) ^ 1, ERR_SLOT);
            if (!ok) break;
            if (elected) {
              if (rank == 0) mbar_expect_tx(bar(&ctrl.k_land[g]), 2 * C::PER * QK_BLOCK);
              for (int c = g * C::PER; c < (g + 1) * C::PER; ++c)
                load_pair(sK + c * QK_BLOCK, &p.mk, 64 * c, 0, tok, of_leader(bar(&ctrl.k_land[g])));
            }
          }
        }
      }
    } else if (warp == WARP_LOAD_V) {
      // ======================= V ============================================================
      const uint32_t elected = elect_one();
      int n = 0;
      while (ok && w.next()) {
        for (int i = 0; i < w.count && ok; ++i, ++n) {
          const int tok = (w.first + i) * TILE;
          for (int h = 0; h < 2; ++h) {
            wait(&ctrl.v_empty[h], (n & 1) ^ 1, ERR_SLOT);
            if (!ok) break;
            if (elected) {
              if (rank == 0) mbar_expect_tx(bar(&ctrl.v_land[h]), 4 * V_BLOCK);
              for (int c = 0; c < 2; ++c)
                load_pair(sV + (2 * h + c) * V_BLOCK, &p.mv, 256 * h + 128 * rank + 64 * c, 0, tok, of_leader(bar(&ctrl.v_land[h])));
            }
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
      const uint32_t elected = elect_one();
      int n = 0, seg = 0;
      while (ok && w.next()) {
        wait(&ctrl.q_land, seg & 1, ERR_Q);
        ++seg;
        const int count = __shfl_sync(0xffffffffu, w.count, 0);
#pragma unroll 1
        for (int i = 0; i < count && ok; ++i, ++n) {
          wait(&ctrl.s_free[n & 1], ((n >> 1) & 1) ^ 1, ERR_FREE);
          const uint32_t tS = t0 + 64 * (n & 1);
#pragma unroll
          for (int g = 0; g < C::GROUPS; ++g) {
            wait(&ctrl.k_land[g], n & 1, ERR_K);
            if (!ok) break;
            tc_fence_after_sync();
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
      const uint32_t elected = elect_one();
      int n = 0, seg = 0;
      while (ok && w.next()) {
        wait(&ctrl.o_free, (seg & 1) ^ 1, ERR_FREE);     // the segment before has been read out
        ++seg;
        const int count = __shfl_sync(0xffffffffu, w.count, 0);
#pragma unroll 1
        for (int i = 0; i < count && ok; ++i, ++n) {
          wait(&ctrl.p_full, n & 1, ERR_P);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            wait(&ctrl.v_land[h], n & 1, ERR_V);
            if (!ok) break;
            tc_fence_after_sync();
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
    while (w.next()) {
      if (tid < ROWS) ctrl.ref[tid] = -INFINITY;
      bar_sync(BAR_BOTH, SOFTMAX_THREADS);
      float m_ref = -INFINITY, l = 0.f;            // l is relative to m_ref
      const uint2* bits = reinterpret_cast<const uint2*>(p.valid) + w.first * 2 + half;
      const int mine = (n & 1) == group ? 0 : 1;   // this group's first tile of the segment
      uint2 ahead = make_uint2(0u, 0u);
      if (mine < w.count) ahead = __ldg(bits + 2 * mine);
      const int n0 = n;                            // tiles of the segments before
#pragma unroll 1
      for (int i = mine; i < w.count; i += 2) {
        n = n0 + i;
        const uint2 seen = ahead;
        if (i + 2 < w.count) ahead = __ldg(bits + 2 * (i + 2));
        wait(&ctrl.s_full[group], (n >> 1) & 1, ERR_S);
        tc_fence_after_sync();
        uint32_t x[64];
        tmem_ld32(tmem + lanes + COL_S + 64 * group, x);
        tmem_ld32(tmem + lanes + COL_S + 64 * group + 32, x + 32);
        tmem_ld_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) arrive_leader(bar(&ctrl.s_free[group]));
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
            alpha = ex2(ref - both);               // 0 for the first
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
          l *= ex2(m_ref - ref);
          m_ref = ref;
        }
        const float sub = ref == -INFINITY ? 0.f : ref;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t pk[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const float a = ex2(fmaf(__uint_as_float(x[2 * k]), c, -sub));
          const float b = ex2(fmaf(__uint_as_float(x[2 * k + 1]), c, -sub));
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
        if (lane == 0) arrive_leader(bar(&ctrl.p_full));
      }
      n = n0 + w.count;
      // ---- the segment's partial ------------------------------------------------------------
      bar_sync(BAR_BOTH, SOFTMAX_THREADS);         // every decision has been made
      const float ref = ctrl.ref[r];
      if (ref != m_ref) l *= ex2(m_ref - ref);
      ctrl.part[2 * group + half][r] = l;
      bar_sync(BAR_BOTH, SOFTMAX_THREADS);
      const float total = (ctrl.part[0][r] + ctrl.part[1][r]) + (ctrl.part[2][r] + ctrl.part[3][r]);
      wait(&ctrl.o_done[(n - 1) & 1], ((n - 1) >> 1) & 1, ERR_O);
      tc_fence_after_sync();
      const bool fail = *reinterpret_cast<volatile int*>(&ctrl.fail) != 0;
      const int row = w.block * 2 * ROWS + rank * ROWS + r;
      const bool none = total == 0.f;
      const float f = none ? 0.f : 1.f / total;
      if (group == 0 && half == 0 && row < p.rows) {
        p.lse_accum[static_cast<int64_t>(w.set) * p.rows + row] = fail ? NAN : none ? -INFINITY : logf(total) + ref * LN2;
        if (w.last)
          for (int s = w.set + 1; s < p.sets; ++s) p.lse_accum[static_cast<int64_t>(s) * p.rows + row] = -INFINITY;
      }
      // each group writes the 256 columns of one product
      float* dst = p.o_accum + (static_cast<int64_t>(w.set) * p.rows + row) * D_V + group * 256 + half * 128;
#pragma unroll 1
      for (int k = 0; k < 4; ++k) {
        uint32_t o[32];
        tmem_ld32(tmem + lanes + COL_O + 128 * group + 32 * k, o);             // warp-collective
        tmem_ld_wait();
        if (k == 3) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) arrive_leader(bar(&ctrl.o_free));
        }
        if (row < p.rows && !fail) {
#pragma unroll
          for (int q = 0; q < 32; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * f);
#pragma unroll
          for (int q = 0; q < 32; q += 8)
            st_global_32(dst + 32 * k + q, o[q], o[q + 1], o[q + 2], o[q + 3], o[q + 4], o[q + 5], o[q + 6], o[q + 7]);
        }
      }
    }
    // no tile at all: nobody else writes the sets of these rows
    if (w.tiles == 0) {
      const int clusters = gridDim.x >> 1;
      for (int64_t i = static_cast<int64_t>(blockIdx.x) * SOFTMAX_THREADS + tid; i < static_cast<int64_t>(p.sets) * p.rows;
           i += static_cast<int64_t>(2 * clusters) * SOFTMAX_THREADS)
        p.lse_accum[i] = -INFINITY;
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

// One launch for what the attention kernels read besides the cache.  CTAs [0, row_ctas): FP8 rows
// of the prefix -> BF16 rows [tokens, d_qk], and a bit per token that says whether it exists; rows
// that do not are zero.  Whole tiles of 128 tokens are written.  Bound by memory: 644 (584) B in
// and 1152 (1024) B out per token; a warp has four tokens in flight.  CTAs [row_ctas, +list_ctas):
// token indices of the prefix.  The others: one query token's list each, of its own tokens or of
// the prefix and those.  List entries behind a length are not written: nothing reads them.
template <int FMT>
__global__ void __launch_bounds__(256)
shared_setup_kernel(const Dsv4SharedPrefixArgs a, const SharedSetup out, const FastDiv page, int row_ctas, int list_ctas) {
  using T = KvTraits<FMT>;
  grid_dependency_wait();
  const int prefix = a.prefix_pages > 0 ? min(max(*a.prefix_length, 0), a.prefix_pages * a.page_block_size) : 0;
  const int n_tok = a.num_blocks * a.page_block_size;
  auto entry = [&](const int32_t* table, int pages, int pos) {
    const int s = slot_of(table, pages, page, pos);
    return s < n_tok ? s : -1;
  };
  if (static_cast<int>(blockIdx.x) >= row_ctas) {
    int x = blockIdx.x - row_ctas;
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

  const int tok0 = blockIdx.x * 32;
  if (tok0 >= (prefix + TILE - 1) / TILE * TILE) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // every warp knows where the CTA's 32 tokens live: lane i looks up token i
  const int tok = tok0 + lane;
  const int col = static_cast<int>(div_by(static_cast<uint32_t>(tok), page));
  int id = -1;
  if (tok < prefix) id = __ldg(a.prefix_table + col);
  const bool live = id >= 0 && id < a.num_blocks;
  const uint32_t word = __ballot_sync(0xffffffffu, live);
  if (threadIdx.x == 0) out.valid[blockIdx.x] = word;
  const int off = tok - col * a.page_block_size;

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
    uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out.rows) + static_cast<int64_t>(tok0 + warp * 4 + k) * T::D_QK);
    if (lane < T::D_NOPE / 16) {
      const ScalePair c = scale_pair(scale[k]);
      const bool two = scale[k] > MAX_ONE_MULTIPLY_SCALE;
      uint32_t o[8];
      dequant4(latent[k].x, c, two, o[0], o[1]);
      dequant4(latent[k].y, c, two, o[2], o[3]);
      dequant4(latent[k].z, c, two, o[4], o[5]);
      dequant4(latent[k].w, c, two, o[6], o[7]);
      dst[2 * lane] = make_uint4(o[0], o[1], o[2], o[3]);
      dst[2 * lane + 1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
    if (lane < 8) dst[T::D_NOPE / 8 + lane] = rope[k];
  }
}

// Joins few partial sets of many rows: one warp per (row, head), which has the whole 2 KB of four
// sets in flight; sets in order, so that the result does not depend on timing.
__global__ void __launch_bounds__(256)
join_sets_kernel(const Dsv4CombineArgs a) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(a.n_rows) * a.h_q;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (item >= rows) return;
  const int row = static_cast<int>(item / a.h_q), h = static_cast<int>(item - static_cast<int64_t>(row) * a.h_q);
  float e = -INFINITY;
  if (lane < a.n_splits) e = a.lse_accum[lane * rows + item];
  const bool failed = __any_sync(0xffffffffu, e != e);
  float m = e;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (failed) m = NAN;
  const float w = e == -INFINITY ? 0.f : expf(e - m);
  float l = w;
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
  for (int s0 = 0; s0 < a.n_splits; s0 += 4) {
    float4 v[4][4];
    float ws[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      ws[j] = s0 + j < a.n_splits ? __shfl_sync(0xffffffffu, w, s0 + j) : 0.f;
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

constexpr int MAX_DEVICES = 64;
std::mutex g_prefix_mu;

template <int DQK>
cudaError_t launch_attn(const PrefixParams& p, int clusters, cudaStream_t st) {
  constexpr size_t smem = prefix_smem_bytes<DQK>();
  static bool configured[MAX_DEVICES] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e) return e;
  if (dev < 0 || dev >= MAX_DEVICES) return cudaErrorInvalidDevice;
  {
    std::lock_guard<std::mutex> lk(g_prefix_mu);
    if (!configured[dev]) {
      e = cudaFuncSetAttribute(prefix_attn_kernel<DQK>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
      if (e) return e;
      configured[dev] = true;
    }
  }
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

// A share is at least line / clusters long, so at most clusters / blocks of them lie in a row
// block, and two more reach into it.
int prefix_attn_sets(int64_t rows, int num_sms) {
  const int64_t blocks = (rows + 2 * ROWS - 1) / (2 * ROWS), clusters = num_sms / 2;
  return static_cast<int>((clusters + blocks - 1) / blocks + 1);
}

int64_t prefix_attn_workspace(int64_t tokens, int d_qk) {
  const int64_t padded = round_up(tokens, TILE);
  return round_up(padded / 8, 256) + padded * d_qk * 2;
}

void prefix_attn_place(int64_t tokens, void* workspace, SharedSetup& out) {
  out.valid = static_cast<uint32_t*>(workspace);
  out.rows = static_cast<uint8_t*>(workspace) + round_up(round_up(tokens, TILE) / 8, 256);
}

cudaError_t launch_shared_setup(const Dsv4SharedPrefixArgs& a, const SharedSetup& out, cudaStream_t st) {
  const int64_t tokens = static_cast<int64_t>(a.prefix_pages) * a.page_block_size;
  const int row_ctas = out.rows != nullptr ? static_cast<int>(round_up(tokens, TILE) / 32) : 0;
  const int list_ctas = out.prefix_list == nullptr ? 0 : static_cast<int>(tokens < 64 * 1024 ? (tokens + 1023) / 1024 : 64);
  const int lists = out.suffix_lists != nullptr || out.joined != nullptr ? a.b * a.s_q : 0;
  if (row_ctas + list_ctas + lists == 0) return cudaSuccess;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(row_ctas) + list_ctas + lists);
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

cudaError_t launch_prefix_attn(const Dsv4SharedPrefixArgs& a, const SharedSetup& setup, int num_sms, cudaStream_t st) {
  const int64_t tokens = static_cast<int64_t>(a.prefix_pages) * a.page_block_size, padded = round_up(tokens, TILE);
  cudaError_t e;
  PrefixParams p;
  p.rows = a.b * a.s_q * a.h_q;
  p.sets = prefix_attn_sets(p.rows, num_sms);
  p.max_tokens = static_cast<int>(tokens);
  p.length = a.prefix_length;
  p.valid = setup.valid;
  p.sm_scale = a.sm_scale;
  p.o_accum = a.o_accum;
  p.lse_accum = a.lse_accum;
  if ((e = make_map_16bit(&p.mq, true, a.q, p.rows, 1, a.d_qk, a.d_qk, a.d_qk, ROWS, 1))) return e;
  if ((e = make_map_16bit(&p.mk, true, setup.rows, static_cast<int>(padded), 1, a.d_qk, a.d_qk, a.d_qk, ROWS, 1))) return e;
  if ((e = make_map_16bit(&p.mv, true, setup.rows, static_cast<int>(padded), 1, a.d_qk, a.d_qk, a.d_qk, TILE, 1))) return e;
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
