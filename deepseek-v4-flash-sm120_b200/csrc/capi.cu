// extern "C" entry points: argument validation, translation to the kernel-side
// parameter block, dispatch.  Allocates nothing and never synchronises.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>

#include "attn_params.cuh"
#include "launchers.h"

namespace {

thread_local char g_cuda_err[256] = "";

int cuda_fail(cudaError_t e) {
  std::snprintf(g_cuda_err, sizeof(g_cuda_err), "%s: %s", cudaGetErrorName(e),
                cudaGetErrorString(e));
  return DSV4_ERR_CUDA;
}

struct DevInfo { int major = 0, minor = 0, sms = 0; bool ok = false; };
constexpr int MAX_DEVICES = 64;
DevInfo g_dev[MAX_DEVICES];
std::mutex g_dev_mu;

int device_info(int device, DevInfo& out) {
  if (device < 0 || device >= MAX_DEVICES) return DSV4_ERR_SHAPE;
  std::lock_guard<std::mutex> lk(g_dev_mu);
  DevInfo& d = g_dev[device];
  if (!d.ok) {
    cudaError_t e;
    if ((e = cudaDeviceGetAttribute(&d.major, cudaDevAttrComputeCapabilityMajor, device)) ||
        (e = cudaDeviceGetAttribute(&d.minor, cudaDevAttrComputeCapabilityMinor, device)) ||
        (e = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, device)))
      return cuda_fail(e);
    d.ok = true;
  }
  out = d;
  return DSV4_OK;
}

int current_device_is_sm100() {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e) return cuda_fail(e);
  DevInfo d;
  int rc = device_info(dev, d);
  if (rc) return rc;
  if (d.major != 10 && std::getenv("DSV4_KERNEL_FORCE") == nullptr) return DSV4_ERR_ARCH;
  return DSV4_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// Largest count that a kernel steps through: room for the strides that its 32-bit counters are
// advanced and rounded by.
constexpr int MOST_ITEMS = 0x7fffffff - 0xffff;
bool aligned32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31u) == 0; }

int check_paged(int kv_format, int d_qk, int page_block, int64_t stride_block, const void* kv) {
  int per_tok;
  if (kv_format == DSV4_KV_MODEL1) { per_tok = 584; if (d_qk != 512) return DSV4_ERR_LAYOUT; }
  else if (kv_format == DSV4_KV_V32) { per_tok = 644; if (d_qk != 576) return DSV4_ERR_LAYOUT; }
  else return DSV4_ERR_LAYOUT;
  if (page_block < 1) return DSV4_ERR_SHAPE;
  if (stride_block < static_cast<int64_t>(page_block) * per_tok) return DSV4_ERR_LAYOUT;
  if ((stride_block & 15) || !aligned16(kv)) return DSV4_ERR_ALIGN;
  return DSV4_OK;
}

long long* g_timeline = nullptr;

int log2_or_minus1(int v) {
  if (v <= 0 || (v & (v - 1))) return -1;
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}

bool want_simple(int flags) {
  if (flags & DSV4_FLAG_IMPL_SIMPLE) return true;
  const char* e = std::getenv("DSV4_IMPL");
  return e && std::strcmp(e, "simple") == 0;
}

}  // namespace

extern "C" {

int dsv4_abi_version(void) { return DSV4_ABI_VERSION; }

const char* dsv4_last_cuda_error(void) { return g_cuda_err; }

const char* dsv4_strerror(int s) {
  switch (s) {
    case DSV4_OK: return "ok";
    case DSV4_ERR_NULL: return "a required pointer is null";
    case DSV4_ERR_SHAPE: return "a size is outside the supported range";
    case DSV4_ERR_LAYOUT: return "d_qk, KV format and page stride do not describe a supported cache layout";
    case DSV4_ERR_ALIGN: return "a pointer or stride is not 16-byte aligned";
    case DSV4_ERR_ARCH: return "the current device is not compute capability 10.x (set DSV4_KERNEL_FORCE to override)";
    case DSV4_ERR_CUDA: return "a CUDA runtime call failed";
    case DSV4_ERR_SCRATCH: return "this split count leaves partials: o_accum and lse_accum are needed";
    case DSV4_ERR_UNSUPPORTED: return "this request is valid but not implemented by this build";
    case DSV4_ERR_SCRATCH_TOO_LARGE: return "split-KV partials exceed the built-in scratch of dsv4_sparse_decode_noalloc (partial sets * b * s_q * h_q * 512 > DSV4_NOALLOC_MAX_O_FLOATS)";
    default: return "unknown status";
  }
}

int dsv4_device_info(int device, int* major, int* minor, int* num_sms) {
  DevInfo d;
  int rc = device_info(device, d);
  if (rc) return rc;
  if (major) *major = d.major;
  if (minor) *minor = d.minor;
  if (num_sms) *num_sms = d.sms;
  return DSV4_OK;
}

int dsv4_plan_splits(int b, int s_q, int h_q, int topk, int extra_topk, int num_sms) {
  if (b < 1 || s_q < 1 || h_q < 1 || topk < 1 || num_sms < 1) return 1;
  const int tile = 128;   // rows one CTA consumes per pipeline step
  const long base = static_cast<long>(b) * s_q * ((h_q + 63) / 64);
  const int tiles = (topk + std::max(extra_topk, 0) + tile - 1) / tile;
  if (base >= num_sms || tiles <= 1) return 1;
  // Cost of a plan in tile-times: waves of CTAs, each walking its tiles plus a
  // fixed prologue/epilogue; a split plan pays one more pass for the combine.
  const double fixed = 0.75, combine = 0.6;
  int best = 1;
  double best_cost = 1e30;
  const int max_s = std::min({tiles, dsv4::combine_max_splits(), 128});
  for (int s = 1; s <= max_s; ++s) {
    const int per = (tiles + s - 1) / s;
    if (s > 1 && (s - 1) * per >= tiles) continue;          // last split would be empty
    const long ctas = base * s;
    const long waves = (ctas + num_sms - 1) / num_sms;
    double cost = waves * (per + fixed) + (s > 1 ? combine + 0.02 * s : 0.0);
    if (cost < best_cost - 1e-9) { best_cost = cost; best = s; }
  }
  return best;
}

int dsv4_split_combine(const Dsv4CombineArgs* a, void* stream) {
  if (!a || !a->o_accum || !a->lse_accum || !a->out || !a->lse) return DSV4_ERR_NULL;
  if (a->n_rows < 0 || a->s_q < 1 || a->h_q < 1 || a->n_splits < 1 ||
      a->n_splits > dsv4::combine_max_splits())
    return DSV4_ERR_SHAPE;
  if (!aligned16(a->o_accum) || (reinterpret_cast<uintptr_t>(a->out) & 7u) ||
      (a->stride_o_b & 3) || (a->stride_o_s & 3) || (a->stride_o_h & 3))
    return DSV4_ERR_ALIGN;
  if (a->n_rows == 0) return DSV4_OK;
  cudaError_t e = dsv4::launch_combine(*a, static_cast<cudaStream_t>(stream));
  return e ? cuda_fail(e) : DSV4_OK;
}

// Splits merged on chip by one thread-block cluster of the tensor-core kernel.  The merge
// pays when it makes the output final (no partials through L2, no combine launch): measured
// on B200, two splits per request (b = 64) gain 8 % per call, whereas merging 8 splits in
// groups of 2 or 4 and still combining the groups loses 9-11 %.  So: the whole request in one
// cluster when n_splits is 2 or 4 (clusters of 4 CTAs with this kernel's shared-memory
// footprint still fill the GPU, clusters of 8 do not), otherwise no cluster.
// DSV4_CLUSTER=1 turns clusters off; DSV4_CLUSTER=group forces groups of 2 or 4 for any
// n_splits they divide (measurement hook).
static int cluster_size_for(int n_splits, bool simple_impl) {
  if (simple_impl || n_splits < 2) return 1;
  static const int mode = [] {
    const char* e = std::getenv("DSV4_CLUSTER");
    if (!e) return 0;
    if (!std::strcmp(e, "group")) return 2;
    return std::atoi(e) == 1 ? 1 : 0;
  }();
  if (mode == 1) return 1;
  if (mode == 2) return (n_splits % 4 == 0) ? 4 : (n_splits % 2 == 0) ? 2 : 1;
  return (n_splits == 2 || n_splits == 4) ? n_splits : 1;
}

int dsv4_decode_partial_sets(const Dsv4DecodeArgs* a) {
  if (!a || a->n_splits < 1) return 0;
  const bool simple = want_simple(a->flags) || !dsv4::sm100_attn_supported(a->kv_format, a->d_qk);
  return a->n_splits / cluster_size_for(a->n_splits, simple);
}

int dsv4_sparse_decode(const Dsv4DecodeArgs* a, void* stream) {
  if (!a || !a->q || !a->kv || !a->indices || !a->out || !a->lse) return DSV4_ERR_NULL;
  if (a->b < 0 || a->s_q < 1 || a->h_q < 1 || a->topk < 1 || a->num_blocks < 1 ||
      a->n_splits < 1 || a->n_splits > dsv4::combine_max_splits() || a->d_v != dsv4::D_V)
    return DSV4_ERR_SHAPE;
  int rc = check_paged(a->kv_format, a->d_qk, a->page_block_size, a->stride_kv_block, a->kv);
  if (rc) return rc;
  if (a->extra_kv) {
    if (!a->extra_indices) return DSV4_ERR_NULL;
    if (a->extra_topk < 1 || a->extra_num_blocks < 1) return DSV4_ERR_SHAPE;
    rc = check_paged(a->kv_format, a->d_qk, a->extra_page_block_size, a->stride_extra_kv_block,
                     a->extra_kv);
    if (rc) return rc;
  }
  if (!aligned16(a->q) || (a->stride_q_b & 7) || (a->stride_q_s & 7) || (a->stride_q_h & 7) ||
      !aligned16(a->out) || (a->stride_o_b & 7) || (a->stride_o_s & 7) || (a->stride_o_h & 7))
    return DSV4_ERR_ALIGN;
  // Scratch is needed only when partials really leave the chip (see dsv4_decode_partial_sets).
  if (dsv4_decode_partial_sets(a) > 1) {
    if (!a->o_accum || !a->lse_accum) return DSV4_ERR_SCRATCH;
    if (!aligned16(a->o_accum)) return DSV4_ERR_ALIGN;
  }
  if ((rc = current_device_is_sm100())) return rc;
  if (a->b == 0) return DSV4_OK;

  dsv4::AttnParams p{};
  p.n_req = a->b * a->s_q;
  p.s_q = a->s_q;
  p.h_q = a->h_q;
  p.topk = a->topk;
  p.extra_topk = a->extra_kv ? a->extra_topk : 0;
  p.n_splits = a->n_splits;
  const bool simple = want_simple(a->flags) || !dsv4::sm100_attn_supported(a->kv_format, a->d_qk);
  p.cluster = cluster_size_for(a->n_splits, simple);
  const int partial_sets = a->n_splits / p.cluster;
  p.flags = a->flags;
  p.mode = dsv4::MODE_DECODE;
  p.page_block = a->page_block_size;
  p.n_tok = a->num_blocks * a->page_block_size;
  p.extra_page_block = a->extra_kv ? a->extra_page_block_size : 1;
  p.extra_n_tok = a->extra_kv ? a->extra_num_blocks * a->extra_page_block_size : 0;
  p.page_shift = log2_or_minus1(p.page_block);
  p.extra_page_shift = log2_or_minus1(p.extra_page_block);
  p.sm_scale = a->sm_scale;
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.kv = static_cast<const uint8_t*>(a->kv);
  p.extra_kv = static_cast<const uint8_t*>(a->extra_kv);
  p.indices = a->indices;
  p.extra_indices = a->extra_kv ? a->extra_indices : nullptr;
  p.topk_length = a->topk_length;
  p.extra_topk_length = a->extra_kv ? a->extra_topk_length : nullptr;
  p.sink = a->attn_sink;
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.lse = a->lse;
  p.max_logits = nullptr;
  p.o_accum = a->o_accum;
  p.lse_accum = a->lse_accum;
  p.stride_q_b = a->stride_q_b; p.stride_q_s = a->stride_q_s; p.stride_q_h = a->stride_q_h;
  p.stride_kv = a->stride_kv_block; p.stride_extra_kv = a->stride_extra_kv_block;
  p.stride_idx_b = a->stride_indices_b; p.stride_idx_s = a->stride_indices_s;
  p.stride_xidx_b = a->stride_extra_indices_b; p.stride_xidx_s = a->stride_extra_indices_s;
  p.stride_o_b = a->stride_o_b; p.stride_o_s = a->stride_o_s; p.stride_o_h = a->stride_o_h;
  p.stride_lse_b = a->stride_lse_b; p.stride_lse_s = a->stride_lse_s; p.stride_lse_h = a->stride_lse_h;
  p.prof = g_timeline;

  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (simple)
    e = dsv4::launch_simple_attn(p, a->kv_format, a->d_qk, st);
  else
    e = dsv4::launch_sm100_attn(p, a->kv_format, a->d_qk, st);
  if (e) return cuda_fail(e);
  if (partial_sets > 1 && !(a->flags & DSV4_FLAG_NO_COMBINE)) {
    Dsv4CombineArgs c{};
    c.n_rows = p.n_req; c.s_q = a->s_q; c.h_q = a->h_q; c.n_splits = partial_sets;
    c.o_accum = a->o_accum; c.lse_accum = a->lse_accum; c.attn_sink = a->attn_sink;
    c.out = a->out; c.lse = a->lse;
    c.stride_o_b = a->stride_o_b; c.stride_o_s = a->stride_o_s; c.stride_o_h = a->stride_o_h;
    c.stride_lse_b = a->stride_lse_b; c.stride_lse_s = a->stride_lse_s; c.stride_lse_h = a->stride_lse_h;
    if ((e = dsv4::launch_combine(c, st))) return cuda_fail(e);
  }
  return DSV4_OK;
}

int dsv4_sparse_prefill(const Dsv4PrefillArgs* a, void* stream) {
  if (!a || !a->q || !a->kv || !a->indices || !a->out || !a->max_logits || !a->lse)
    return DSV4_ERR_NULL;
  if (a->s_q < 0 || a->s_kv < 0 || a->h_q < 1 || a->topk < 1 || a->d_v != dsv4::D_V)
    return DSV4_ERR_SHAPE;
  int rc;
  if (a->kv_format == DSV4_KV_BF16) {
    if (a->d_qk != 512 && a->d_qk != 576) return DSV4_ERR_LAYOUT;
    if (!aligned16(a->kv) || (a->stride_kv_row & 7)) return DSV4_ERR_ALIGN;
  } else {
    if ((rc = check_paged(a->kv_format, a->d_qk, a->page_block_size, a->stride_kv_row, a->kv)))
      return rc;
    if (a->num_blocks < 1) return DSV4_ERR_SHAPE;
  }
  if (!aligned16(a->q) || (a->stride_q_s & 7) || (a->stride_q_h & 7) || !aligned16(a->out) ||
      (a->stride_o_s & 7) || (a->stride_o_h & 7))
    return DSV4_ERR_ALIGN;
  if ((rc = current_device_is_sm100())) return rc;
  if (a->s_q == 0) return DSV4_OK;

  dsv4::AttnParams p{};
  p.n_req = a->s_q;
  p.s_q = 1;
  p.h_q = a->h_q;
  p.topk = a->topk;
  p.n_splits = 1;
  p.cluster = 1;
  p.flags = a->flags;
  p.mode = dsv4::MODE_PREFILL;
  p.page_block = a->kv_format == DSV4_KV_BF16 ? 1 : a->page_block_size;
  p.n_tok = a->kv_format == DSV4_KV_BF16 ? a->s_kv : a->num_blocks * a->page_block_size;
  p.extra_page_block = 1;
  p.page_shift = log2_or_minus1(p.page_block);
  p.extra_page_shift = 0;
  p.sm_scale = a->sm_scale;
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.kv = static_cast<const uint8_t*>(a->kv);
  p.indices = a->indices;
  p.topk_length = a->topk_length;
  p.sink = a->attn_sink;
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.lse = a->lse;
  p.max_logits = a->max_logits;
  p.stride_q_b = a->stride_q_s; p.stride_q_h = a->stride_q_h;
  p.stride_kv = a->stride_kv_row;
  p.stride_idx_b = a->stride_indices_s;
  p.stride_o_b = a->stride_o_s; p.stride_o_h = a->stride_o_h;
  p.stride_lse_b = a->stride_lse_s; p.stride_lse_h = 1;
  p.stride_ml_b = a->stride_ml_s;
  p.prof = g_timeline;

  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (want_simple(a->flags) || !dsv4::sm100_attn_supported(a->kv_format, a->d_qk))
    e = dsv4::launch_simple_attn(p, a->kv_format, a->d_qk, st);
  else
    e = dsv4::launch_sm100_attn(p, a->kv_format, a->d_qk, st);
  return e ? cuda_fail(e) : DSV4_OK;
}

// How a shared-prefix decode is done, and its scratch.
//   JOINED  one list per query token, of the prefix and its own tokens, for the sparse kernel:
//           reads the prefix once per request, but is two or three short launches;
//   DENSE   the prefix by launch_prefix_attn, with the own tokens where their table is not too
//           wide, else those by the sparse kernel, joined;
//   LISTS   the same with the prefix by the sparse kernel too, as one list for all rows.
// Scratch is sized by one call and used by another, so the plan depends on the sizes alone: it is
// made for the 148 SMs of a B200 whatever the device has (the kernels take any number of sets).
constexpr int PLAN_SMS = 148;
// DENSE keeps 2 d_qk bytes of workspace for every token that the prefix table can hold, in each
// captured graph too.
constexpr int64_t DENSE_MOST_BYTES = 4ll << 30;
enum SharedForm { FORM_JOINED, FORM_DENSE, FORM_LISTS };
struct SharedPlan {
  SharedForm form;
  bool own;                                // DENSE: the own tokens in the same pass
  int prefix_sets, suffix_splits;          // partial sets of the two parts (JOINED: splits in the second)
  int64_t prefix_bytes, suffix_bytes;      // of the workspace: the prefix's part, then the lists
};
static SharedForm choose_form(const Dsv4SharedPrefixArgs* a, int64_t rows, int64_t plen, int64_t slen) {
  const bool by_list = a->prefix_splits > 0 || a->suffix_splits > 0 || want_simple(a->flags);
  if (by_list || plen + slen == 0 || (a->flags & DSV4_FLAG_SHARED_LISTS)) return FORM_LISTS;
  if (plen == 0 || (a->flags & DSV4_FLAG_SHARED_JOINED)) return FORM_JOINED;
  if ((a->flags & DSV4_FLAG_SHARED_DENSE) && dsv4::prefix_attn_fits(*a, false)) return FORM_DENSE;
  // JOINED up to 4 tiles of 128 tokens an SM, half as many where they are of more than 32 heads, and
  // lists of 4000 tokens (microseconds, JOINED / DENSE / LISTS, prefix x query tokens x heads: 2000 x
  // 4 x 16: 19 / 25 / 35; 512 x 57 x 20, 456 tiles: 21 / 29 / 33; 6000 x 16 x 8, 768 tiles: 41 / 31 /
  // 35; 2000 x 3 x 64: 23 / 29 / 37; 1088 x 32 x 64, 288 tiles: 39 / 31 / 50; 16000 x 1 x 16: 31 / 26 /
  // 31).  Over 200 drawn calls of up to 60 requests and 30000 tokens the rules here cost 0.8 % over
  // the best form of each.
  const int64_t tiles = static_cast<int64_t>(a->b) * a->s_q * ((a->h_q + 63) / 64) * ((plen + slen + 127) / 128);
  if (tiles * (a->h_q <= 32 ? 1 : 2) <= 4ll * PLAN_SMS && plen + slen <= 4000) return FORM_JOINED;
  // LISTS for up to 64 rows behind a long prefix: converting it all costs more than reading its FP8
  // rows once (1 x 16, 16000: 26 DENSE, 31 LISTS; 65536: 54 and 43; 262144: 154 and 98; two blocks of
  // rows, 2 x 64, 65536: 58 and 68).
  if (rows <= 64 && plen > 40000) return FORM_LISTS;
  // DENSE for all others, unless its workspace passes what a caller can be expected to have: tables
  // of more than 3.7 million tokens (d_qk 576) go by LISTS, 4 bytes a token (64 x 64 behind 4194304
  // tokens: 29 ms DENSE with 4.8 GB, 72 LISTS with 17 MB; 16 x 64: 7.9 and 19).
  return dsv4::prefix_attn_fits(*a, false) && dsv4::prefix_attn_workspace(*a, false) <= DENSE_MOST_BYTES ? FORM_DENSE : FORM_LISTS;
}

static SharedPlan plan_shared(const Dsv4SharedPrefixArgs* a) {
  SharedPlan p{};
  const int64_t rows = static_cast<int64_t>(a->b) * a->s_q * a->h_q;
  const int64_t plen = static_cast<int64_t>(a->prefix_pages) * a->page_block_size;
  const int64_t slen = static_cast<int64_t>(a->max_pages) * a->page_block_size;
  const int64_t tokens = static_cast<int64_t>(a->b) * a->s_q;
  p.form = choose_form(a, rows, plen, slen);
  if (p.form == FORM_JOINED) {
    p.suffix_splits = dsv4_plan_splits(a->b, a->s_q, a->h_q, static_cast<int>(plen + slen), 0, PLAN_SMS);
    p.suffix_bytes = (tokens * (plen + slen) + a->b) * 4;
    return p;
  }
  if (p.form == FORM_DENSE) {
    // In the same pass the own tokens are converted to BF16 rows like the prefix's, which pays while
    // those rows stay in L2, up to 131072 tokens that the table can hold; and a tile of them is of use
    // to its request's rows alone: fewer where those are less than an eighth of a block's 128
    // (microseconds, same pass / own launch; requests x heads, prefix, own: 64 x 64, 32768, 64 to
    // 2048: 219 / 244; 64 x 64, 2048, 64 to 2048: 61 / 91; 16 x 128, 8192, 4096 to 8192: 101 / 135; 64
    // x 16, 8192, 64 to 512: 53 / 58; 27 x 8, 10976, up to 1056: 37 / 45.  Beyond: 64 x 16, 32768, 1024
    // to 2048: 130 / 121; 64 x 64, 8192, 2048 to 4096: 168 / 162; 256 x 64, 1024, 1100: 217 / 184;
    // 128 x 8, 32768, 64 to 512: 108 / 102).
    const int64_t most_own = a->s_q * a->h_q >= 16 ? 131072 : 49152;
    p.own = slen > 0 && a->b * ((slen + 127) / 128 * 128) <= most_own && dsv4::prefix_attn_fits(*a, true);
    p.prefix_sets = dsv4::prefix_attn_sets(rows, PLAN_SMS);
    p.prefix_bytes = dsv4::prefix_attn_workspace(*a, p.own);
    if (p.own) return p;
  } else if (plen > 0) {
    p.prefix_sets = a->prefix_splits > 0 ? a->prefix_splits
                                         : dsv4_plan_splits(1, 1, static_cast<int>(rows), static_cast<int>(plen), 0, PLAN_SMS);
    p.prefix_bytes = (plen + 63) / 64 * 64 * 4;
  }
  if (slen > 0)
    p.suffix_splits = a->suffix_splits > 0 ? a->suffix_splits
                                           : dsv4_plan_splits(a->b, a->s_q, a->h_q, static_cast<int>(slen), 0, PLAN_SMS);
  p.suffix_bytes = slen * tokens * 4;
  return p;
}

static int check_shared(const Dsv4SharedPrefixArgs* a) {
  if (!a) return DSV4_ERR_NULL;
  if (a->b < 0 || a->s_q < 1 || a->h_q < 1 || a->num_blocks < 1 || a->page_block_size < 1 || a->d_v != dsv4::D_V ||
      !(a->sm_scale > 0.0f) || !(a->sm_scale <= 1.0e38f) || a->prefix_pages < 0 || a->max_pages < 0 || a->prefix_splits < 0 || a->suffix_splits < 0 ||
      a->prefix_splits > 64 || a->suffix_splits > 64)
    return DSV4_ERR_SHAPE;
  const int64_t most = MOST_ITEMS;
  if (static_cast<int64_t>(a->num_blocks) * a->page_block_size > most ||
      static_cast<int64_t>(a->prefix_pages) * a->page_block_size > most ||
      static_cast<int64_t>(a->max_pages) * a->page_block_size > most ||
      (static_cast<int64_t>(a->prefix_pages) + a->max_pages) * a->page_block_size > most ||
      static_cast<int64_t>(a->b) * a->s_q > most / a->h_q ||
      static_cast<int64_t>(a->b) * a->s_q * a->h_q > 64ll * 65535)
    return DSV4_ERR_SHAPE;
  // grid dimensions: heads of the combine, and rows as heads of the cross-check kernel
  if (a->h_q > 65535 || (want_simple(a->flags) && static_cast<int64_t>(a->b) * a->s_q * a->h_q > 65535))
    return DSV4_ERR_SHAPE;
  return DSV4_OK;
}

int dsv4_shared_prefix_scratch(const Dsv4SharedPrefixArgs* a, int num_sms, int32_t* sets, int64_t* bytes) {
  int rc = check_shared(a);
  if (rc) return rc;
  if (!sets || !bytes) return DSV4_ERR_NULL;
  if (num_sms < 2) return DSV4_ERR_SHAPE;
  *sets = 0;
  *bytes = 0;
  if (a->b == 0) return DSV4_OK;         // (the plan divides by the rows' blocks)
  const SharedPlan p = plan_shared(a);
  *sets = p.prefix_sets + p.suffix_splits;
  if (p.form == FORM_JOINED && p.suffix_splits == 1) *sets = 0;      // final at once
  *bytes = p.prefix_bytes + p.suffix_bytes;
  return DSV4_OK;
}

int dsv4_shared_prefix_decode(const Dsv4SharedPrefixArgs* a, void* stream) {
  int rc = check_shared(a);
  if (rc) return rc;
  if (!a->q || !a->kv || !a->out || !a->lse || (a->prefix_pages && (!a->prefix_table || !a->prefix_length)) ||
      (a->max_pages && (!a->block_table || !a->suffix_length)))
    return DSV4_ERR_NULL;
  if ((rc = check_paged(a->kv_format, a->d_qk, a->page_block_size, a->stride_kv_block, a->kv))) return rc;
  if (a->max_pages && a->stride_table < 0) return DSV4_ERR_SHAPE;
  if (!aligned16(a->q) || !aligned16(a->out) || (a->stride_o_b & 7) || (a->stride_o_s & 7) || (a->stride_o_h & 7))
    return DSV4_ERR_ALIGN;
  if ((rc = current_device_is_sm100())) return rc;
  if (a->b == 0) return DSV4_OK;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e) return cuda_fail(e);
  DevInfo info;
  if ((rc = device_info(dev, info))) return rc;
  const SharedPlan plan = plan_shared(a);
  const int sets = plan.prefix_sets + plan.suffix_splits;
  if (sets > 0 && (plan.form != FORM_JOINED || sets > 1)) {
    if (!a->o_accum || !a->lse_accum) return DSV4_ERR_SCRATCH;
    if (!aligned32(a->o_accum)) return DSV4_ERR_ALIGN;
  }
  if (plan.prefix_bytes + plan.suffix_bytes > 0) {
    if (!a->workspace) return DSV4_ERR_SCRATCH;
    if (!aligned32(a->workspace)) return DSV4_ERR_ALIGN;
  }
  const int64_t rows = static_cast<int64_t>(a->b) * a->s_q * a->h_q;
  const int64_t plen = static_cast<int64_t>(a->prefix_pages) * a->page_block_size;
  const int64_t slen = static_cast<int64_t>(a->max_pages) * a->page_block_size;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int32_t* lists = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(a->workspace) + plan.prefix_bytes);
  dsv4::SharedSetup setup{};
  if (plan.form == FORM_DENSE) dsv4::prefix_attn_place(*a, plan.own, setup);
  if (plan.form == FORM_LISTS && plen > 0) setup.prefix_list = static_cast<int32_t*>(a->workspace);
  if (plan.form == FORM_JOINED) {
    setup.joined = lists;
    setup.lens = lists + static_cast<int64_t>(a->b) * a->s_q * (plen + slen);
  } else if (slen > 0 && !plan.own) {
    setup.suffix_lists = lists;
  }
  if ((e = dsv4::launch_shared_setup(*a, setup, st))) return cuda_fail(e);

  if (plan.form == FORM_JOINED) {
    Dsv4DecodeArgs d{};
    d.b = a->b; d.s_q = a->s_q; d.h_q = a->h_q; d.d_qk = a->d_qk; d.d_v = a->d_v;
    d.topk = static_cast<int>(plen + slen);
    d.kv_format = a->kv_format; d.num_blocks = a->num_blocks; d.page_block_size = a->page_block_size;
    d.n_splits = plan.suffix_splits;
    d.flags = DSV4_FLAG_MASK_INVALID | DSV4_FLAG_ZERO_LENGTH_EMPTY;
    d.sm_scale = a->sm_scale;
    d.q = a->q; d.kv = a->kv; d.indices = setup.joined; d.topk_length = setup.lens; d.attn_sink = a->attn_sink;
    d.out = a->out; d.lse = a->lse; d.o_accum = a->o_accum; d.lse_accum = a->lse_accum;
    d.stride_q_h = a->d_qk;
    d.stride_q_s = static_cast<int64_t>(a->h_q) * a->d_qk;
    d.stride_q_b = d.stride_q_s * a->s_q;
    d.stride_kv_block = a->stride_kv_block;
    d.stride_indices_s = d.topk;
    d.stride_indices_b = static_cast<int64_t>(d.topk) * a->s_q;
    d.stride_o_b = a->stride_o_b; d.stride_o_s = a->stride_o_s; d.stride_o_h = a->stride_o_h;
    d.stride_lse_b = a->stride_lse_b; d.stride_lse_s = a->stride_lse_s; d.stride_lse_h = a->stride_lse_h;
    return dsv4_sparse_decode(&d, stream);
  }
  if (plan.form == FORM_DENSE && (e = dsv4::launch_prefix_attn(*a, setup, plan.prefix_sets, info.sms, st))) return cuda_fail(e);

  dsv4::AttnParams p{};
  p.cluster = 1;
  p.keep_partials = 1;
  p.flags = DSV4_FLAG_MASK_INVALID | DSV4_FLAG_ZERO_LENGTH_EMPTY;
  p.mode = dsv4::MODE_DECODE;
  p.page_block = a->page_block_size;
  p.n_tok = a->num_blocks * a->page_block_size;
  p.extra_page_block = 1;
  p.page_shift = log2_or_minus1(p.page_block);
  p.sm_scale = a->sm_scale;
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.kv = static_cast<const uint8_t*>(a->kv);
  p.stride_kv = a->stride_kv_block;
  p.stride_q_h = a->d_qk;
  p.out = static_cast<__nv_bfloat16*>(a->out);
  p.lse = a->lse;
  auto attend = [&]() {
    return want_simple(a->flags) ? dsv4::launch_simple_attn(p, a->kv_format, a->d_qk, st)
                                 : dsv4::launch_sm100_attn(p, a->kv_format, a->d_qk, st);
  };
  if (plan.prefix_sets > 0 && plan.form == FORM_LISTS) {
    // the rows of all requests as the heads of one: each block of 64 rows walks the prefix once
    p.n_req = p.s_q = 1;
    p.h_q = static_cast<int>(rows);
    p.topk = a->prefix_pages * a->page_block_size;
    p.n_splits = plan.prefix_sets;
    p.indices = setup.prefix_list;
    p.topk_length = a->prefix_length;
    p.o_accum = a->o_accum;
    p.lse_accum = a->lse_accum;
    if ((e = attend())) return cuda_fail(e);
  }
  if (plan.suffix_splits > 0) {
    p.n_req = a->b * a->s_q;
    p.s_q = a->s_q;
    p.h_q = a->h_q;
    p.topk = a->max_pages * a->page_block_size;
    p.n_splits = plan.suffix_splits;
    p.indices = setup.suffix_lists;
    p.topk_length = a->suffix_length;
    p.stride_q_s = static_cast<int64_t>(a->h_q) * a->d_qk;
    p.stride_q_b = p.stride_q_s * a->s_q;
    p.stride_idx_s = p.topk;
    p.stride_idx_b = static_cast<int64_t>(p.topk) * a->s_q;
    p.o_accum = a->o_accum + plan.prefix_sets * rows * dsv4::D_V;
    p.lse_accum = a->lse_accum + plan.prefix_sets * rows;
    if ((e = attend())) return cuda_fail(e);
  }
  Dsv4CombineArgs c{};
  c.n_rows = a->b * a->s_q; c.s_q = a->s_q; c.h_q = a->h_q; c.n_splits = sets;
  c.o_accum = a->o_accum; c.lse_accum = a->lse_accum; c.attn_sink = a->attn_sink;
  c.out = a->out; c.lse = a->lse;
  c.stride_o_b = a->stride_o_b; c.stride_o_s = a->stride_o_s; c.stride_o_h = a->stride_o_h;
  c.stride_lse_b = a->stride_lse_b; c.stride_lse_s = a->stride_lse_s; c.stride_lse_h = a->stride_lse_h;
  e = dsv4::launch_join_sets(c, st);
  return e ? cuda_fail(e) : DSV4_OK;
}

int dsv4_plan_dense_splits(int t_q, int t_k, int b, int h_q, int h_kv, int num_sms) {
  if (t_q < 1 || t_k < 1 || b < 1 || h_q < 1 || h_kv < 1 || h_q % h_kv || num_sms < 1) return 1;
  const int64_t ctas = dsv4::dense_ctas(t_q, b, h_q, h_kv);
  const double tiles = static_cast<double>(t_k) / b / 128.0;           // of a sequence, on average
  if (tiles <= 2.0) return 1;
  // In microseconds, fitted to calls of 1 to 200 sequences on a B200: a CTA starts and ends in 5,
  // streams a tile of 128 keys in 1 (64 to 80 KB, what its buffers keep in flight), and the
  // GPU's memory gives a tile in 0.0105; a launch more costs 3, a range 0.6, and the partials are
  // written and read at 4 TB/s.  The lengths are on the device: the longest sequence is taken to
  // be eight times the average one.  (One sequence of 8000 keys, 64 heads on one: 78 us uncut, 22
  // in ranges; 60 of 1 to 20000 keys, 8 heads of 64: 170 and 81; 32 of 4096, 32 heads on 8, which
  // fill the GPU evenly: 95 and 102.)
  const double total = static_cast<double>(t_k) / 128.0;
  const double longest = std::fmin(tiles * 8.0, total);
  const double line = ctas * tiles, memory = line * 0.0105;
  const double uncut = std::fmax(5.0 + longest, std::fmax((ctas * 5.0 + line) / num_sms, memory));
  const double per = std::fmax(line / num_sms, std::sqrt(0.6 * longest));      // tiles of a range
  const double used = ctas * std::fmax(tiles / per, 1.0);
  const double partials = 2.0 * t_q * h_q * 128.0 * 4.0 * (tiles / per + 1.0) / 4.0e6;
  const double cut = std::fmax(5.0 + per, std::fmax((used * 5.0 + line) / num_sms, memory + 5.0)) + 3.0 + 0.6 * longest / per + partials;
  if (cut >= uncut) return 1;
  return static_cast<int>(std::fmin(std::fmax(longest / per, 2.0), dsv4::DENSE_MAX_SPLITS));
}

int dsv4_dense_prefill(const Dsv4DensePrefillArgs* a, void* stream) {
  if (!a) return DSV4_ERR_NULL;
  if (a->b < 0 || a->t_q < 0 || a->t_k < 0 || a->t_q > MOST_ITEMS || a->t_k > MOST_ITEMS || a->h_q < 1 || a->h_kv < 1 || a->h_q % a->h_kv ||
      a->n_splits < 1 || a->n_splits > dsv4::DENSE_MAX_SPLITS || !(a->sm_scale > 0.0f) ||
      !(a->sm_scale <= 1.0e38f) || dsv4::dense_ctas(a->t_q, a->b, a->h_q, a->h_kv) > (a->n_splits > 1 ? 1 << 24 : 0x7fffffff))
    return DSV4_ERR_SHAPE;
  if (!((a->d_qk == 64 && a->d_v == 64) || (a->d_qk == 128 && a->d_v == 128) ||
        (a->d_qk == 192 && a->d_v == 128)))
    return DSV4_ERR_LAYOUT;
  if (a->dtype != DSV4_DTYPE_BF16 && a->dtype != DSV4_DTYPE_FP16) return DSV4_ERR_UNSUPPORTED;
  if (a->b == 0 || a->t_q == 0) return DSV4_OK;
  if (!a->q || !a->cu_seqlens_q || !a->cu_seqlens_k || !a->out || !a->max_logits || !a->lse ||
      (a->t_k && (!a->k || !a->v)))
    return DSV4_ERR_NULL;
  struct { const void* p; int64_t t, h; int nt, nh; } views[4] = {
      {a->q, a->stride_q_t, a->stride_q_h, a->t_q, a->h_q},
      {a->k, a->stride_k_t, a->stride_k_h, a->t_k, a->h_kv},
      {a->v, a->stride_v_t, a->stride_v_h, a->t_k, a->h_kv},
      {a->out, a->stride_o_t, a->stride_o_h, a->t_q, a->h_q}};
  for (const auto& v : views) {
    if (v.nt == 0) continue;
    if (!aligned16(v.p)) return DSV4_ERR_ALIGN;
    if (v.nt > 1 && (v.t < 1 || (v.t & 7) || v.t >= (1ll << 38))) return DSV4_ERR_ALIGN;
    if (v.nh > 1 && (v.h < 1 || (v.h & 7) || v.h >= (1ll << 38))) return DSV4_ERR_ALIGN;
  }
  if (a->n_splits > 1) {
    if (!a->o_accum || !a->stat_accum) return DSV4_ERR_SCRATCH;
    if (!aligned32(a->o_accum) || (reinterpret_cast<uintptr_t>(a->stat_accum) & 7u)) return DSV4_ERR_ALIGN;
  }
  int rc = current_device_is_sm100();
  if (rc) return rc;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e) return cuda_fail(e);
  DevInfo info;
  if ((rc = device_info(dev, info))) return rc;
  e = dsv4::launch_dense_prefill(*a, info.sms, static_cast<cudaStream_t>(stream));
  return e ? cuda_fail(e) : DSV4_OK;
}

int dsv4_kv_store(const Dsv4StoreArgs* a, void* stream) {
  if (!a || !a->k_nope || !a->k_rope || !a->slots || !a->kv) return DSV4_ERR_NULL;
  if (a->n_tokens < 0 || a->num_blocks < 1 || a->page_block_size < 1) return DSV4_ERR_SHAPE;
  const int d_qk = a->kv_format == DSV4_KV_MODEL1 ? 512 : 576;
  int rc = check_paged(a->kv_format, d_qk, a->page_block_size, a->stride_kv_block, a->kv);
  if (rc) return rc;
  if (!aligned16(a->k_nope) || !aligned16(a->k_rope) || (a->stride_nope & 7) || (a->stride_rope & 7))
    return DSV4_ERR_ALIGN;
  cudaError_t e = dsv4::launch_kv_store(*a, nullptr, static_cast<cudaStream_t>(stream));
  return e ? cuda_fail(e) : DSV4_OK;
}

int dsv4_kv_store_rows(const Dsv4StoreRowsArgs* r, void* stream) {
  if (!r || !r->k || !r->loc || !r->kv) return DSV4_ERR_NULL;
  if (r->n_tokens < 0 || r->num_blocks < 1 || r->page_block_size < 1) return DSV4_ERR_SHAPE;
  if (r->kv_format != DSV4_KV_MODEL1 && r->kv_format != DSV4_KV_V32) return DSV4_ERR_LAYOUT;
  const int d_qk = r->kv_format == DSV4_KV_MODEL1 ? 512 : 576;
  int rc = check_paged(r->kv_format, d_qk, r->page_block_size, r->stride_kv_block, r->kv);
  if (rc) return rc;
  // the RoPE values start d_qk - 64 elements into the row: 896 / 1024 bytes, a multiple of 16
  if (!aligned16(r->k) || (r->stride_k & 7) || r->stride_k < d_qk) return DSV4_ERR_ALIGN;
  Dsv4StoreArgs a{};
  a.n_tokens = r->n_tokens; a.kv_format = r->kv_format;
  a.num_blocks = r->num_blocks; a.page_block_size = r->page_block_size;
  a.k_nope = r->k;
  a.k_rope = static_cast<const uint16_t*>(r->k) + (d_qk - 64);
  a.stride_nope = a.stride_rope = r->stride_k;
  a.kv = r->kv; a.stride_kv_block = r->stride_kv_block;
  a.slots = r->loc_is_int64 ? static_cast<const int64_t*>(r->loc) : nullptr;
  const int32_t* loc32 = r->loc_is_int64 ? nullptr : static_cast<const int32_t*>(r->loc);
  cudaError_t e = dsv4::launch_kv_store(a, loc32, static_cast<cudaStream_t>(stream));
  return e ? cuda_fail(e) : DSV4_OK;
}

int dsv4_build_slot_maps(const Dsv4SlotMapArgs* a, void* stream) {
  if (!a || !a->cu_new || !a->cu_total || !a->n_taken) return DSV4_ERR_NULL;
  if (a->b < 0 || a->b > dsv4::SLOT_MAP_MAX_REQUESTS || a->max_pages < 0 || a->page_block_size < 1 ||
      a->n_slots < 0 || a->n_free < 0)
    return DSV4_ERR_SHAPE;
  if ((a->b && (!a->cached_lens || !a->new_lens)) || (a->b && a->max_pages && !a->block_table) ||
      (a->n_free && !a->free_pages) || (a->n_slots && (!a->slots || !a->positions)))
    return DSV4_ERR_NULL;
  if (a->b > 1 && a->stride_table < a->max_pages) return DSV4_ERR_LAYOUT;   // rows would overlap
  int rc = current_device_is_sm100();
  if (rc) return rc;
  cudaError_t e = dsv4::launch_slot_maps(*a, static_cast<cudaStream_t>(stream));
  return e ? cuda_fail(e) : DSV4_OK;
}

int dsv4_page_indices(const Dsv4PageIndicesArgs* a, void* stream) {
  if (!a) return DSV4_ERR_NULL;
  if (a->n_rows < 0 || a->topk < 0 || a->n_rows > MOST_ITEMS || a->topk > MOST_ITEMS || a->b < 0 || a->max_pages < 0 || a->page_block_size < 1 ||
      a->s_q < 1 || a->stride_positions < 0 || a->stride_table < 0)
    return DSV4_ERR_SHAPE;
  if (a->n_rows == 0 || a->topk == 0) return DSV4_OK;
  if (!a->positions || !a->indices || (a->b && a->max_pages && !a->block_table)) return DSV4_ERR_NULL;
  int rc = current_device_is_sm100();
  if (rc) return rc;
  cudaError_t e = dsv4::launch_page_indices(*a, static_cast<cudaStream_t>(stream));
  return e ? cuda_fail(e) : DSV4_OK;
}

int dsv4_gather_dequant(const void* kv, int64_t stride_kv_block, int32_t kv_format,
                        int32_t num_blocks, int32_t page_block_size, const int32_t* indices,
                        int32_t n, void* rows_bf16, int32_t method, void* stream) {
  if (!kv || !indices || !rows_bf16) return DSV4_ERR_NULL;
  if (n < 0 || num_blocks < 1) return DSV4_ERR_SHAPE;
  const int d_qk = kv_format == DSV4_KV_MODEL1 ? 512 : 576;
  int rc = check_paged(kv_format, d_qk, page_block_size, stride_kv_block, kv);
  if (rc) return rc;
  if (!aligned16(rows_bf16)) return DSV4_ERR_ALIGN;
  cudaError_t e = dsv4::launch_gather_dequant(kv, stride_kv_block, kv_format, num_blocks,
                                              page_block_size, indices, n, rows_bf16, method,
                                              static_cast<cudaStream_t>(stream));
  return e ? cuda_fail(e) : DSV4_OK;
}

int dsv4_debug_set_timeline(void* device_buffer) {
  g_timeline = static_cast<long long*>(device_buffer);
  return DSV4_OK;
}

int dsv4_device_status(int32_t* status_out, int reset) {
  if (!status_out) return DSV4_ERR_NULL;
  int v = 0;
  cudaError_t e = dsv4::read_attn_error(&v, reset != 0);
  if (e) return cuda_fail(e);
  int d = 0;
  if ((e = dsv4::read_dense_error(&d, reset != 0))) return cuda_fail(e);
  if (v == 0) v = d;
  if ((e = dsv4::read_prefix_error(&d, reset != 0))) return cuda_fail(e);
  if (v == 0) v = d;
  *status_out = v;
  return DSV4_OK;
}

int dsv4_gather_heads(const Dsv4GatherArgs* a, void* stream) {
  if (!a || !a->out_local || !a->lse_local || !a->counter || !a->status) return DSV4_ERR_NULL;
  if (a->world < 1 || a->world > DSV4_MAX_PEERS || a->rank < 0 || a->rank >= a->world || a->b < 0 ||
      a->s_q < 1 || a->h_local < 1)
    return DSV4_ERR_SHAPE;
  for (int r = 0; r < a->world; ++r) {
    if (!a->peer_out[r] || !a->peer_lse[r] || !a->peer_flags[r]) return DSV4_ERR_NULL;
    if (!aligned16(a->peer_out[r])) return DSV4_ERR_ALIGN;
  }
  if (!aligned16(a->out_local)) return DSV4_ERR_ALIGN;
  cudaError_t e = dsv4::launch_gather_heads(*a, static_cast<cudaStream_t>(stream));
  return e ? cuda_fail(e) : DSV4_OK;
}

int dsv4_sparse_decode_gather(const Dsv4DecodeArgs* d, const Dsv4GatherArgs* g, void* stream) {
  if (!d || !g || !g->counter || !g->status || !d->out || !d->lse) return DSV4_ERR_NULL;
  if (g->world < 1 || g->world > DSV4_MAX_PEERS || g->rank < 0 || g->rank >= g->world ||
      g->b != d->b || g->s_q != d->s_q || g->h_local != d->h_q)
    return DSV4_ERR_SHAPE;
  for (int r = 0; r < g->world; ++r) {
    if (!g->peer_out[r] || !g->peer_lse[r] || !g->peer_flags[r]) return DSV4_ERR_NULL;
    if (!aligned16(g->peer_out[r])) return DSV4_ERR_ALIGN;
  }
  // the local result must be dense: it is what the exchange kernel reads
  if (d->stride_o_h != 512 || d->stride_o_s != static_cast<int64_t>(d->h_q) * 512 ||
      d->stride_o_b != static_cast<int64_t>(d->s_q) * d->h_q * 512 || d->stride_lse_s != 1 ||
      d->stride_lse_h != d->s_q || d->stride_lse_b != static_cast<int64_t>(d->h_q) * d->s_q)
    return DSV4_ERR_LAYOUT;
  // Decode (with its split combine, when the plan has one) and the exchange kernel behind it
  // with programmatic dependent launch: the exchange kernel is resident before the rows are
  // final.  A combine step that stored straight into the peers' buffers was measured 1-2 us
  // slower per step than this pair (more CTAs fencing at system scope, narrower NVLink
  // stores), so it was taken out again.
  int rc = dsv4_sparse_decode(d, stream);
  if (rc) return rc;
  Dsv4GatherArgs ga = *g;
  ga.out_local = d->out;
  ga.lse_local = d->lse;
  return dsv4_gather_heads(&ga, stream);
}

int dsv4_umma_selftest(int mode, int n, int k, const void* a, const void* b, float* d,
                       int32_t* status, void* stream) {
  if (!a || !b || !d || !status) return DSV4_ERR_NULL;
  if (mode < 0 || mode > 1 || n < 16 || n > 64 || (n & 15) || k < 64 || k > 256 || (k & 63))
    return DSV4_ERR_SHAPE;
  int rc = current_device_is_sm100();
  if (rc) return rc;
  cudaError_t e = dsv4::launch_umma_selftest(mode, n, k, a, b, d, status,
                                             static_cast<cudaStream_t>(stream));
  return e ? cuda_fail(e) : DSV4_OK;
}

}  // extern "C"
