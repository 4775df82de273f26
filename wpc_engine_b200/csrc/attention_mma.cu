// Entry points of bfloat16 attention over the paged cache on the tensor cores: all earlier
// positions, or a window of them (the kernels are in attention_mma.cuh).
#include "attention_mma.cuh"

using namespace wpc;

extern "C" {

// Decode attention copies pages of earlier positions before the kernel ahead has finished
// (1, the default) or starts every copy after it (0); returns the old setting.
int wpc_attention_decode_early_pages(int on) {
  const int was = fa::early_pages();
  fa::early_pages() = on ? 1 : 0;
  return was;
}

// 1 if these sizes can take the tensor-core kernels, else 0 (the plain kernel takes them).
int wpc_attention_mma_supports(int nh, int nkv, int hd) {
  return hd >= 16 && hd <= 128 && hd % 16 == 0 && nkv >= 1 && nh % nkv == 0 && nh / nkv <= 16;
}

// One query token per sequence: q row b belongs to sequence b (at most 1024 sequences).
// n_ctas CTAs share the pages of all sequences evenly (1..1024).  part_o: float32
// [(n_ctas + B * nkv) * 16 * hd], part_ml: float32 [(n_ctas + B * nkv) * 16 * 2], counters:
// B * nkv tickets that are zero between launches.
int wpc_attention_decode(const void* q, int q_stride, void* out, int out_stride, const void* k_pages,
                         const void* v_pages, const int* page_table, int table_width, const int* ctx_lens, int B,
                         int nh, int nkv, int hd, float scale, int window, int n_ctas, float* part_o,
                         float* part_ml, int* counters, int n_counters, cudaStream_t stream) {
  if (B <= 0) return 0;
  if (!wpc_attention_mma_supports(nh, nkv, hd) || (q_stride % 2) || (out_stride % 2) || B > fa::MAX_DECODE_SEQS)
    return WPC_ERR_UNSUPPORTED;
  if (n_ctas < 1 || n_ctas > 1024 || !part_o || !part_ml || !counters || B * nkv > n_counters)
    return WPC_ERR_BAD_ARGUMENT;
  WPC_DISPATCH_HD(hd, fa::launch_decode<HD, fa::MODE_PLAIN>(q, q_stride, out, out_stride, k_pages, v_pages, page_table, table_width,
                                           ctx_lens, B, nh, nkv, scale, window, n_ctas, part_o, part_ml, counters,
                                           fa::Extra{}, stream));
}

// The same with a thread-block cluster of `cluster` CTAs (2..16) to each (sequence, kv head) pair,
// which share the pair's pages and add up through one another's shared memory; for few pairs
// of about equal lengths.  Needs (nh / nkv) * hd <= 1024 and at most 1024 CTAs.  With groups > 1
// that many clusters share a pair's pages through part_o (float32 [B * nkv * groups * (nh / nkv)
// * hd]), part_ml (float32 [B * nkv * groups * 32]) and B * nkv tickets that are zero between
// launches.
int wpc_attention_decode_cluster(const void* q, int q_stride, void* out, int out_stride, const void* k_pages,
                                 const void* v_pages, const int* page_table, int table_width, const int* ctx_lens,
                                 int B, int nh, int nkv, int hd, float scale, int window, int cluster, int groups,
                                 float* part_o, float* part_ml, int* counters, int n_counters,
                                 cudaStream_t stream) {
  if (B <= 0) return 0;
  if (!wpc_attention_mma_supports(nh, nkv, hd) || (q_stride % 2) || (out_stride % 2) ||
      (nh / nkv) * hd > fa::CLUSTER_DECODE_MAX_OUT)
    return WPC_ERR_UNSUPPORTED;
  if (cluster < 2 || cluster > fa::CLUSTER_DECODE_MAX_RANKS || groups < 1 ||
      groups > fa::CLUSTER_DECODE_MAX_GROUPS || (long)B * nkv * cluster * groups > 1024)
    return WPC_ERR_BAD_ARGUMENT;
  if (groups > 1 && (!part_o || !part_ml || !counters || B * nkv > n_counters)) return WPC_ERR_BAD_ARGUMENT;
  WPC_DISPATCH_HD(hd, fa::launch_decode_cluster<HD, fa::MODE_PLAIN>(q, q_stride, out, out_stride, k_pages, v_pages, page_table,
                                                   table_width, ctx_lens, B, nh, nkv, scale, window, cluster, groups,
                                                   part_o, part_ml, counters, fa::Extra{}, stream));
}

// Clusters of `cluster` CTAs of the cluster decode kernel that run at once: with the short ring
// (two CTAs to an SM) or, `alone`, with the long one.
int wpc_attention_decode_cluster_capacity(int hd, int cluster, int alone) {
  if (cluster < 2 || cluster > fa::CLUSTER_DECODE_MAX_RANKS) return 0;
  if (alone) { WPC_DISPATCH_HD(hd, fa::decode_cluster_capacity<HD, fa::DECODE_STAGES_ALONE>(cluster)); }
  WPC_DISPATCH_HD(hd, fa::decode_cluster_capacity<HD, fa::DECODE_STAGES_SHARED>(cluster));
}

int wpc_attention_prefill(const void* q, int q_stride, void* out, int out_stride, const void* k_pages,
                          const void* v_pages, const int* page_table, int table_width, const int* cu_seqlens,
                          const int* ctx_lens, int B, int max_new, int nh, int nkv, int hd, float scale, int window,
                          cudaStream_t stream) {
  if (B <= 0 || max_new <= 0) return 0;
  if (!wpc_attention_mma_supports(nh, nkv, hd) || (q_stride % 2) || (out_stride % 2)) return WPC_ERR_UNSUPPORTED;
  WPC_DISPATCH_HD(hd, fa::launch_prefill<HD, fa::MODE_PLAIN>(q, q_stride, out, out_stride, k_pages, v_pages, page_table, table_width,
                                            cu_seqlens, ctx_lens, B, max_new, nh, nkv, scale, window, fa::Extra{}, stream));
}

}  // extern "C"
