// Block tables and slot maps on the GPU: what a serving step derives from its request
// lengths before it can write or read the paged cache.
//
// slot_maps_kernel.  With c_r tokens of request r cached, n_r new ones and P tokens a page,
//   old_r = ceil(c_r / P), need_r = ceil((c_r + n_r) / P) - old_r,
//   start_r / first_r = exclusive sums of n_r / need_r over the requests,
// page j >= old_r of request r is free_pages[first_r + j - old_r], and new token t of the
// packed batch (request r: start_r <= t < start_r + n_r) sits at position c_r + t - start_r.
// Bound by latency, not by bytes (12 B a token): lengths -> sums -> request of a token ->
// page id are dependent steps.  So ONE launch does all of it: every CTA sums the lengths
// itself (8 B a request out of L2, cheaper than a second launch or a grid-wide hand-over),
// keeps both sums in shared memory and finds its tokens' requests by bisection there.  A new
// page's id comes from the free list in both places that need it (its table entry and its
// tokens' slots), so no CTA reads an entry another one writes.  Measured: 64 requests of one token
// 2.7 us in a graph; 301 prompts of 1 to 2048 tokens: 7 us from cold caches (launch, and four
// dependent reads of about 0.8 us).
//
// page_indices_kernel.  slot = table[r][pos / P] * P + pos % P per list entry: 4 B in, 4 B
// out, bound by memory for prefill lists.  16-byte loads and stores where rows allow, the
// division by a multiplication prepared on the host.  Measured: 8192 x 2048 entries 23.7 us,
// 5.7 TB/s (0.87 of a copy's rate); 64 x 2048 entries 2.7 us in a graph.
#include "attn_params.cuh"
#include "launch_util.h"
#include "launchers.h"
#include "paging.cuh"

namespace dsv4 {
namespace {

constexpr int SLOT_THREADS = 512;
constexpr int MAX_I32 = 0x7fffffff;

__device__ __forceinline__ int saturate(long long v) {
  return v > MAX_I32 ? MAX_I32 : static_cast<int>(v);
}

__device__ __forceinline__ long long warp_inclusive(long long v, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// Largest r in [0, n) with a[r] <= x; a[0] = 0, ascending.  Entries of empty requests are
// equal to their successor's, so the last of equals is the request that holds x.
__device__ __forceinline__ int last_not_above(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Pages of the first `tokens` tokens, at most `width`.  Two lengths add up to less than
// 2^32, so positions and token counts of one request are unsigned 32-bit numbers.
__device__ __forceinline__ int pages_of(uint32_t tokens, uint32_t page, int width) {
  const uint32_t p = tokens / page + (tokens % page != 0);
  return p < static_cast<uint32_t>(width) ? static_cast<int>(p) : width;
}

__global__ void __launch_bounds__(SLOT_THREADS)
slot_maps_kernel(const Dsv4SlotMapArgs a) {
  extern __shared__ int sums[];                 // start[b + 1], first[b + 1]
  int* start = sums;
  int* first = sums + a.b + 1;
  __shared__ long long part[3][SLOT_THREADS / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int WARPS = SLOT_THREADS / 32;
  grid_dependency_wait();

  long long carry_new = 0, carry_need = 0, carry_all = 0;
  for (int r0 = 0; r0 < a.b; r0 += SLOT_THREADS) {
    const int r = r0 + tid;
    int c = 0, n = 0, need = 0;
    if (r < a.b) {
      c = max(a.cached_lens[r], 0);
      n = max(a.new_lens[r], 0);
      need = pages_of(static_cast<uint32_t>(c) + n, a.page_block_size, a.max_pages) -
             pages_of(c, a.page_block_size, a.max_pages);
    }
    const long long all = static_cast<long long>(c) + n;
    const long long i_new = warp_inclusive(n, lane), i_need = warp_inclusive(need, lane);
    const long long i_all = warp_inclusive(all, lane);
    if (lane == 31) { part[0][warp] = i_new; part[1][warp] = i_need; part[2][warp] = i_all; }
    __syncthreads();
    if (warp < 3) {
      const long long v = warp_inclusive(lane < WARPS ? part[warp][lane] : 0, lane);
      if (lane < WARPS) part[warp][lane] = v;
    }
    __syncthreads();
    const long long b_new = carry_new + (warp ? part[0][warp - 1] : 0);
    const long long b_need = carry_need + (warp ? part[1][warp - 1] : 0);
    const long long b_all = carry_all + (warp ? part[2][warp - 1] : 0);
    if (r < a.b) {
      start[r] = saturate(b_new + i_new - n);
      first[r] = saturate(b_need + i_need - need);
      if (blockIdx.x == 0) {
        a.cu_new[r + 1] = saturate(b_new + i_new);
        a.cu_total[r + 1] = saturate(b_all + i_all);
      }
    }
    carry_new += part[0][WARPS - 1];
    carry_need += part[1][WARPS - 1];
    carry_all += part[2][WARPS - 1];
    __syncthreads();                            // part is rewritten by the next round
  }
  const int total_new = saturate(carry_new), total_need = saturate(carry_need);
  if (blockIdx.x == 0 && tid == 0) {
    a.cu_new[0] = 0;
    a.cu_total[0] = 0;
    *a.n_taken = total_need;
  }
  if (a.b == 0) {
    for (long long t = blockIdx.x * SLOT_THREADS + tid; t < a.n_slots; t += gridDim.x * SLOT_THREADS) {
      a.slots[t] = -1;
      a.positions[t] = -1;
    }
    return;
  }
  __syncthreads();

  // new tokens, then new pages, as one range of work items
  const long long items = static_cast<long long>(a.n_slots) + total_need;
  for (long long it = static_cast<long long>(blockIdx.x) * SLOT_THREADS + tid; it < items;
       it += static_cast<long long>(gridDim.x) * SLOT_THREADS) {
    if (it < a.n_slots) {
      const int t = static_cast<int>(it);
      long long slot = -1;
      int pos = -1;
      if (t < total_new) {
        const int r = last_not_above(start, a.b, t);
        const int c = max(a.cached_lens[r], 0);
        const uint32_t p = static_cast<uint32_t>(c) + (t - start[r]), page = a.page_block_size;
        pos = saturate(p);
        const uint32_t ucol = p / page;
        const int off = static_cast<int>(p - ucol * page);
        if (ucol < static_cast<uint32_t>(a.max_pages)) {
          const int col = static_cast<int>(ucol);
          const int old = pages_of(c, a.page_block_size, a.max_pages);
          int id = -1;
          if (col < old) {
            id = a.block_table[r * a.stride_table + col];
          } else {
            const long long f = static_cast<long long>(first[r]) + (col - old);
            if (f < a.n_free) id = a.free_pages[f];
          }
          if (id >= 0) slot = static_cast<long long>(id) * a.page_block_size + off;
        }
      }
      a.slots[t] = slot;
      a.positions[t] = pos;
    } else {
      const int g = static_cast<int>(it - a.n_slots);
      const int r = last_not_above(first, a.b, g);
      const int old = pages_of(max(a.cached_lens[r], 0), a.page_block_size, a.max_pages);
      const long long col = static_cast<long long>(old) + (g - first[r]);
      if (col < a.max_pages)                    // (always, unless the sums saturated)
        a.block_table[r * a.stride_table + col] = g < a.n_free ? a.free_pages[g] : -1;
    }
  }
}

// threadIdx.x walks a row, threadIdx.y and the grid the rows.
template <bool VEC>
__global__ void __launch_bounds__(256)
page_indices_kernel(const Dsv4PageIndicesArgs a, const FastDiv page) {
  grid_dependency_wait();
  const int row = blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= a.n_rows) return;
  int r = -1;
  if (a.cu_seqlens == nullptr) {
    r = row / a.s_q;
  } else if (a.b > 0 && row >= a.cu_seqlens[0] && row < a.cu_seqlens[a.b]) {
    int lo = 0, hi = a.b;                       // cu[lo] <= row < cu[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu_seqlens[mid] <= row) lo = mid; else hi = mid;
    }
    r = lo;
  }
  const int32_t* table = r >= 0 && r < a.b ? a.block_table + r * a.stride_table : nullptr;
  const int32_t* src = a.positions + row * a.stride_positions;
  int32_t* dst = a.indices + static_cast<int64_t>(row) * a.topk;
  const int width = table ? a.max_pages : 0;
  if (VEC) {
    const int n4 = a.topk >> 2;
    for (int i = threadIdx.x; i < n4; i += 2 * blockDim.x) {
      const int j = i + blockDim.x;
      const int4 p = __ldg(reinterpret_cast<const int4*>(src) + i);
      const int4 q = j < n4 ? __ldg(reinterpret_cast<const int4*>(src) + j) : make_int4(-1, -1, -1, -1);
      reinterpret_cast<int4*>(dst)[i] = make_int4(slot_of(table, width, page, p.x), slot_of(table, width, page, p.y),
                                                  slot_of(table, width, page, p.z), slot_of(table, width, page, p.w));
      if (j < n4)
        reinterpret_cast<int4*>(dst)[j] = make_int4(slot_of(table, width, page, q.x), slot_of(table, width, page, q.y),
                                                    slot_of(table, width, page, q.z), slot_of(table, width, page, q.w));
    }
  } else {
    for (int i = threadIdx.x; i < a.topk; i += blockDim.x) dst[i] = slot_of(table, width, page, src[i]);
  }
}

}  // namespace

cudaError_t launch_slot_maps(const Dsv4SlotMapArgs& a, cudaStream_t st) {
  const size_t smem = 2 * (static_cast<size_t>(a.b) + 1) * sizeof(int);
  int dev = 0, sms = 0;
  cudaError_t e = allow_shared_memory<slot_maps_kernel>(2 * (SLOT_MAP_MAX_REQUESTS + 1) * sizeof(int), &dev);
  if (e) return e;
  if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev))) return e;
  const long long want = (static_cast<long long>(a.n_slots) + a.b + SLOT_THREADS - 1) / SLOT_THREADS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(want < 1 ? 1 : want < sms ? want : sms));
  cfg.blockDim = dim3(SLOT_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  cfg.numAttrs = add_overlap_attribute(attr);
  return cudaLaunchKernelEx(&cfg, slot_maps_kernel, a);
}

cudaError_t launch_page_indices(const Dsv4PageIndicesArgs& a, cudaStream_t st) {
  const bool vec = (a.topk & 3) == 0 && (a.stride_positions & 3) == 0 &&
                   (reinterpret_cast<uintptr_t>(a.positions) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(a.indices) & 15) == 0;
  const int per_row = vec ? (a.topk / 4 + 1) / 2 : a.topk;
  int tx = 32;
  while (tx < per_row && tx < 256) tx <<= 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(tx, 256 / tx);
  cfg.gridDim = dim3((a.n_rows + 256 / tx - 1) / (256 / tx));
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  cfg.numAttrs = add_overlap_attribute(attr);
  const FastDiv page = fast_div(static_cast<uint32_t>(a.page_block_size));
  return vec ? cudaLaunchKernelEx(&cfg, page_indices_kernel<true>, a, page)
             : cudaLaunchKernelEx(&cfg, page_indices_kernel<false>, a, page);
}

}  // namespace dsv4
