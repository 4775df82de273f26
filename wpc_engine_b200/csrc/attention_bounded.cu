// Entry points of bfloat16 attention for sequences longer than their cache, by the forms of the
// kernels in attention_mma.cuh that the ordinary attention does not need:
//
//   sinks   beside the last `window` positions a query sees the first `sinks` ones
//           (scores of all other positions are -inf): the pages of the sinks and of the window are
//           read, nothing between them, so the time goes with window + sinks, whatever the length.
//   sums    all earlier positions, and what the sums of weights need afterwards (attention_sums.cu):
//           a decode step's scaled scores with each row's maximum and inverse sum, or each
//           row's log-sum of a prefill.
//
// Measured (7B shape; 28 heads, 4 KV heads of 128): one sequence at position 24,577, window 4,096, 4 sinks 7.2 us,
// latency (5 pages a CTA); 64 of up to 8,000, window 2,048, 70 sinks 55.0 to 58.5, 268 MB at 4.6 to 4.9 TB/s; with sums 8
// sequences of 4,001 19.5 to 21.7, 67 MB, 17 of it ordinary attention (a second kernel adds up the weights: inside
// the cluster kernel the same took 24.3), one of 32,768 24.4 to 26.5.
#include "attention_mma.cuh"

using namespace wpc;

static int decode_bounded(const void* q, int q_stride, void* out, int out_stride, const void* k_pages,
                          const void* v_pages, const int* page_table, int table_width, const int* ctx_lens,
                          int B, int nh, int nkv, int hd, float scale, int window, int sinks, int n_ctas,
                          int cluster, int groups, float* part_o, float* part_ml, int* counters, int n_counters,
                          float* scores, int score_stride, float* row_ml, int n_pages, cudaStream_t stream) {
  if (B <= 0) return 0;
  if (!wpc_attention_mma_supports(nh, nkv, hd) || (q_stride % 2) || (out_stride % 2)) return WPC_ERR_UNSUPPORTED;
  if (n_pages < 1) return WPC_ERR_BAD_ARGUMENT;
  const bool sums = scores != nullptr;
  if (sums ? (!row_ml || score_stride < 64 || score_stride % 64 || window > 0 || sinks != 0) : (sinks < 1 || window < 1))
    return WPC_ERR_BAD_ARGUMENT;
  const fa::Extra x{sinks, score_stride, scores, (float2*)row_ml, nullptr, n_pages};
  if (cluster) {
    if ((nh / nkv) * hd > fa::CLUSTER_DECODE_MAX_OUT) return WPC_ERR_UNSUPPORTED;
    if (cluster < 2 || cluster > fa::CLUSTER_DECODE_MAX_RANKS || groups < 1 ||
        groups > fa::CLUSTER_DECODE_MAX_GROUPS || (long)B * nkv * cluster * groups > 1024)
      return WPC_ERR_BAD_ARGUMENT;
    if (groups > 1 && (!part_o || !part_ml || !counters || (long)B * nkv > n_counters)) return WPC_ERR_BAD_ARGUMENT;
    if (sums) {
      WPC_DISPATCH_HD(hd, fa::launch_decode_cluster<HD, fa::MODE_SUMS>(
          q, q_stride, out, out_stride, k_pages, v_pages, page_table, table_width, ctx_lens, B, nh, nkv, scale, window,
          cluster, groups, part_o, part_ml, counters, x, stream));
    }
    WPC_DISPATCH_HD(hd, fa::launch_decode_cluster<HD, fa::MODE_SINKS>(
        q, q_stride, out, out_stride, k_pages, v_pages, page_table, table_width, ctx_lens, B, nh, nkv, scale, window,
        cluster, groups, part_o, part_ml, counters, x, stream));
  }
  if (B > fa::MAX_DECODE_SEQS) return WPC_ERR_UNSUPPORTED;
  if (n_ctas < 1 || n_ctas > 1024 || !part_o || !part_ml || !counters || (long)B * nkv > n_counters)
    return WPC_ERR_BAD_ARGUMENT;
  if (sums) {
    WPC_DISPATCH_HD(hd, fa::launch_decode<HD, fa::MODE_SUMS>(
        q, q_stride, out, out_stride, k_pages, v_pages, page_table, table_width, ctx_lens, B, nh, nkv, scale, window,
        n_ctas, part_o, part_ml, counters, x, stream));
  }
  WPC_DISPATCH_HD(hd, fa::launch_decode<HD, fa::MODE_SINKS>(
      q, q_stride, out, out_stride, k_pages, v_pages, page_table, table_width, ctx_lens, B, nh, nkv, scale, window,
      n_ctas, part_o, part_ml, counters, x, stream));
}

extern "C" {

int wpc_attention_decode_bounded(const void* q, int q_stride, void* out, int out_stride, const void* k_pages,
                                 const void* v_pages, const int* page_table, int table_width, const int* ctx_lens,
                                 int B, int nh, int nkv, int hd, float scale, int window, int sinks, int n_ctas,
                                 int cluster, int groups, float* part_o, float* part_ml, int* counters, int n_counters,
                                 float* scores, int score_stride, float* row_ml, const int* token_positions, int max_ctx,
                                 int n_pages, float* weight_sums, int* stored_positions, int* status,
                                 cudaStream_t stream) {
  const int rc = decode_bounded(q, q_stride, out, out_stride, k_pages, v_pages, page_table, table_width, ctx_lens, B, nh,
                                nkv, hd, scale, window, sinks, n_ctas, cluster, groups, part_o, part_ml, counters,
                                n_counters, scores, score_stride, row_ml, n_pages, stream);
  if (rc || !scores) return rc;
  return wpc_weight_sums_decode(scores, score_stride, row_ml, page_table, table_width, ctx_lens, token_positions, B, nh,
                                nkv, max_ctx, n_pages, weight_sums, stored_positions, status, stream);
}

int wpc_attention_prefill_bounded(const void* q, int q_stride, void* out, int out_stride, const void* k_pages,
                                  const void* v_pages, const int* page_table, int table_width, const int* cu_seqlens,
                                  const int* ctx_lens, int B, int max_new, int nh, int nkv, int hd, float scale,
                                  int window, int sinks, float* lse, int n_pages, cudaStream_t stream) {
  if (B <= 0 || max_new <= 0) return 0;
  if (n_pages < 1) return WPC_ERR_BAD_ARGUMENT;
  if (!wpc_attention_mma_supports(nh, nkv, hd) || (q_stride % 2) || (out_stride % 2)) return WPC_ERR_UNSUPPORTED;
  if (lse ? (window > 0 || sinks != 0) : (sinks < 1 || window < 1)) return WPC_ERR_BAD_ARGUMENT;
  const fa::Extra x{sinks, 0, nullptr, nullptr, lse, n_pages};
  if (lse) {
    WPC_DISPATCH_HD(hd, fa::launch_prefill<HD, fa::MODE_SUMS>(q, q_stride, out, out_stride, k_pages, v_pages, page_table,
                                                             table_width, cu_seqlens, ctx_lens, B, max_new, nh, nkv,
                                                             scale, window, x, stream));
  }
  WPC_DISPATCH_HD(hd, fa::launch_prefill<HD, fa::MODE_SINKS>(q, q_stride, out, out_stride, k_pages, v_pages, page_table,
                                                            table_width, cu_seqlens, ctx_lens, B, max_new, nh, nkv,
                                                            scale, window, x, stream));
}

}  // extern "C"
