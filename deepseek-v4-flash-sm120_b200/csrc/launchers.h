// Host-side launch functions implemented by the kernel translation units.
#pragma once

#include <cuda_runtime.h>

#include "dsv4_b200.h"

#include <cstdlib>

namespace dsv4 {

struct AttnParams;

// Programmatic dependent launch: with this attribute a kernel may be set up on the SMs
// while the kernel before it in the stream is still in its last phase; both kernels here
// execute griddepcontrol.wait before their first global access, so they still observe all
// of the predecessor's writes.  DSV4_NO_PDL=1 turns the attribute off.
// Returns the number of attributes written (0 or 1).
inline int add_overlap_attribute(cudaLaunchAttribute* attr) {
  static const bool off = [] {
    const char* e = std::getenv("DSV4_NO_PDL");
    return e != nullptr && e[0] != '\0' && e[0] != '0';
  }();
  if (off) return 0;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  return 1;
}

// CUDA-core cross-check kernels (simple_kernels.cu).
cudaError_t launch_simple_attn(const AttnParams& p, int kv_format, int d_qk, cudaStream_t st);
cudaError_t launch_combine(const Dsv4CombineArgs& a, cudaStream_t st);
int combine_max_splits();
// `slots32` non-null: the slot mapping is int32 and a.slots is ignored.
cudaError_t launch_kv_store(const Dsv4StoreArgs& a, const int32_t* slots32, cudaStream_t st);
cudaError_t launch_gather_dequant(const void* kv, int64_t stride, int kv_format, int num_blocks,
                                  int page_block, const int32_t* indices, int n, void* rows,
                                  int method, cudaStream_t st);

// Block tables and slot maps (paging.cu).
constexpr int SLOT_MAP_MAX_REQUESTS = 16384;     // both sums of a request list in shared memory
cudaError_t launch_slot_maps(const Dsv4SlotMapArgs& a, cudaStream_t st);
cudaError_t launch_page_indices(const Dsv4PageIndicesArgs& a, cudaStream_t st);

// Set-up of a shared-prefix decode (shared_prefix_sm100.cu), one launch: what is not null of
//   rows, valid    the prefix as BF16 rows and, when own_padded is not 0, each request's own
//                  tokens (`padded` rows, then own_padded for each), and a bit per row: it exists,
//   unfit          a bit per row of own tokens: its latent part is not finite, and zeros stand there,
//   starts         where the tiles of the row blocks start (prefix_attn_place sets these six),
//   prefix_list    token indices of the prefix,
//   suffix_lists   of every query token's own tokens, a list of max_pages * page entries each,
//   joined, lens   both one after the other, prefix_pages * page entries more each, and the
//                  requests' list lengths.
struct SharedSetup {
  void* rows;
  uint32_t *valid, *unfit;
  int32_t* starts;
  int padded, own_padded;
  int32_t *prefix_list, *suffix_lists, *joined, *lens;
};
cudaError_t launch_shared_setup(const Dsv4SharedPrefixArgs& a, const SharedSetup& out, cudaStream_t st);
// Joins partial sets of BF16 outputs (like launch_combine, for few sets and many rows).
cudaError_t launch_join_sets(const Dsv4CombineArgs& a, cudaStream_t st);

// Attention of many rows over a shared prefix, into the first `sets` partial sets
// (shared_prefix_sm100.cu); prefix_attn_sets says how many suit a number of SMs, and two or more
// are enough for any.
int prefix_attn_sets(int64_t rows, int num_sms);
// `own`: with the requests' own tokens.  Do the sizes fit, and how many bytes of workspace?
bool prefix_attn_fits(const Dsv4SharedPrefixArgs& a, bool own);
int64_t prefix_attn_workspace(const Dsv4SharedPrefixArgs& a, bool own);
void prefix_attn_place(const Dsv4SharedPrefixArgs& a, bool own, SharedSetup& out);
cudaError_t launch_prefix_attn(const Dsv4SharedPrefixArgs& a, const SharedSetup& rows, int sets, int num_sms, cudaStream_t st);
cudaError_t read_prefix_error(int* value, bool reset);

// Dense attention over packed sequences (dense_attn_sm100.cu).
constexpr int DENSE_MAX_SPLITS = 64;
int64_t dense_ctas(int t_q, int b, int h_q, int h_kv);      // CTAs of one key range, at most
cudaError_t launch_dense_prefill(const Dsv4DensePrefillArgs& a, int num_sms, cudaStream_t st);
cudaError_t read_dense_error(int* value, bool reset);

// tcgen05 kernels (sparse_attn_sm100.cu).  `supported` reports whether the
// tensor-core kernel handles this (format, d_qk) pair.
bool sm100_attn_supported(int kv_format, int d_qk);
cudaError_t launch_sm100_attn(const AttnParams& p, int kv_format, int d_qk, cudaStream_t st);
cudaError_t read_attn_error(int* value, bool reset);
cudaError_t launch_gather_heads(const Dsv4GatherArgs& a, cudaStream_t st);
cudaError_t launch_umma_selftest(int mode, int n, int k, const void* a, const void* b, float* d,
                                 int32_t* status, cudaStream_t st);

}  // namespace dsv4
