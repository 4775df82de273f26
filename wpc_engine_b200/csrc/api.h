// The C interface of the kernel library.  Every function launches on `stream`, allocates
// nothing and returns 0, a cudaError_t value, or one of the WPC_ERR_* codes of common.cuh.
// Element types are named by WPC_DTYPE_F32 (0) and WPC_DTYPE_BF16 (1).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

// Programmatic dependent launch for all kernels of the library: on (1, the default) or off (0).
int wpc_set_pdl(int on);
// 1 if the next kernel of the library on this stream of the current device will not start ahead of the
// one before it (after wpc_move_kept), else 0.
int wpc_pdl_next_waits(cudaStream_t stream);
// How long a kernel waits on one of its mbarriers before it gives up, records
// WPC_ERR_DEVICE_WAIT in the status word it was given and returns (default 2 s).  `starve` = 1
// is for tests of that path: the kernels with TMA producers start no copies, so their waits
// run out; nothing else about them changes.  2: the same, but in the kernel of prompts' weight
// sums in every other CTA only.
int wpc_set_wait_policy(unsigned long long limit_ns, int starve);

int wpc_embed(const int* tokens, const void* table, int table_dtype, float* out, int T, int H, int V,
              cudaStream_t stream);
// rows == null: out [T, H]; else out [n_rows, H], row i the norm of x[rows[i]]
int wpc_rmsnorm(const float* x, const float* gain, float eps, void* out, int out_dtype, int T, int H,
                const int* rows, int n_rows, cudaStream_t stream);
// out[t, i] = act(gate) * up; act: WPC_ACT_SILU (1) or WPC_ACT_GELU_TANH (2) of common.cuh
int wpc_gate_mul(const void* gu, void* out, int dtype, int T, int I, int group, int act, cudaStream_t stream);
int wpc_add(float* x, const void* y, int y_dtype, size_t n, cudaStream_t stream);
int wpc_gather_rows(const float* x, const int* idx, float* out, int n_rows, int H, int T, cudaStream_t stream);
int wpc_convert(const void* in, int in_dtype, void* out, int out_dtype, size_t n, cudaStream_t stream);
int wpc_rope_angles(const int* positions, const double* inv_freq, float* cosv, float* sinv, int T, int R,
                    cudaStream_t stream);
// interleaved = 0: pairs (r, r + hd/2); 1: pairs (2r, 2r + 1)
int wpc_rope_inplace(void* x, int dtype, int row_stride, int T, int n_heads, int hd, int R, const float* cosv,
                     const float* sinv, int interleaved, cudaStream_t stream);
// RMS norm with gain [hd] of each of the first n_heads heads of every row, in place
int wpc_head_rmsnorm(void* x, int dtype, int row_stride, int T, int n_heads, int hd, const float* gain, float eps,
                     cudaStream_t stream);
int wpc_qk_rope_kv_store(void* qkv, int dtype, int row_stride, int T, int nh, int nkv, int hd, int R,
                         const float* cosv, const float* sinv, void* k_pages, void* v_pages,
                         const int* page_table, int table_width, const int* seq_of_token, const int* positions,
                         int n_pages, int* status, cudaStream_t stream);
int wpc_fill_normal(void* out, int dtype, size_t n, uint64_t key, float mean, float std, cudaStream_t stream);

int wpc_gemm_simt(const void* A, int a_dtype, int lda, const void* W, int w_dtype, int ldw, const float* bias,
                  void* C, int out_dtype, int ldc, int accumulate, int M, int N, int K, cudaStream_t stream);

int wpc_gemm_tc_set_stage_limit(int limit);
int wpc_gemm_tc_workspace(int rows_a, int rows_b, int bn, int splits, size_t* scratch_floats, int* n_counters);
int wpc_gemm_tc(const void* a, int lda, int rows_a, const void* b, int ldb, int rows_b, int K, const float* bias,
                void* out, int out_dtype, int ldc, int accumulate, int gated, int swap, int bn, int splits,
                float* scratch, size_t scratch_floats, int* counters, int n_counters, int* status,
                int prefetch_weights, int tall, int cluster, cudaStream_t stream);
int wpc_gemm_tc_cluster_capacity(int bn, int splits);
int wpc_gemm_tc_rope_store(const void* w, int ldw, const void* x, int ldx, int tokens, int K, const float* bias, void* out,
                           int ldc, int bn, int splits, int prefetch_weights, int nh, int nkv, int hd, int R,
                           const float* cosv, const float* sinv, void* k_pages, void* v_pages, const int* page_table,
                           int table_width, const int* seq_of_token, const int* positions, int n_pages, int* status,
                           cudaStream_t stream);

// sinks: the first positions that a query sees beside its window (0 without a window);
// lse: null, or [T][nh] for each row's maximum + log2(sum) of its scores in units of log 2
int wpc_attention_plain_bounded(const void* q, int q_stride, void* out, int out_stride, int dtype,
                                const void* k_pages, const void* v_pages, const int* page_table, int table_width,
                                const int* seq_of_token, const int* positions, int T, int nh, int nkv, int hd,
                                float scale, int window, int sinks, int n_splits, float* part, float* lse, int n_pages,
                                cudaStream_t stream);

int wpc_attention_mma_supports(int nh, int nkv, int hd);
int wpc_attention_decode_early_pages(int on);
int wpc_attention_decode(const void* q, int q_stride, void* out, int out_stride, const void* k_pages,
                         const void* v_pages, const int* page_table, int table_width, const int* ctx_lens, int B,
                         int nh, int nkv, int hd, float scale, int window, int n_ctas, float* part_o, float* part_ml,
                         int* counters, int n_counters, cudaStream_t stream);
int wpc_attention_decode_cluster_capacity(int hd, int cluster, int alone);
int wpc_attention_decode_cluster(const void* q, int q_stride, void* out, int out_stride, const void* k_pages,
                                 const void* v_pages, const int* page_table, int table_width, const int* ctx_lens,
                                 int B, int nh, int nkv, int hd, float scale, int window, int cluster, int groups,
                                 float* part_o, float* part_ml, int* counters, int n_counters,
                                 cudaStream_t stream);
int wpc_attention_prefill(const void* q, int q_stride, void* out, int out_stride, const void* k_pages,
                          const void* v_pages, const int* page_table, int table_width, const int* cu_seqlens,
                          const int* ctx_lens, int B, int max_new, int nh, int nkv, int hd, float scale, int window,
                          cudaStream_t stream);

int wpc_attention_prefill_tc_supports(int nh, int nkv, int hd);
int wpc_attention_prefill_tc(const void* q, int q_stride, void* out, int out_stride, const void* k_pages,
                             const void* v_pages, const int* page_table, int table_width, const int* cu_seqlens,
                             const int* ctx_lens, int B, int max_new, int nh, int nkv, int hd, float scale,
                             int window, int* status, int n_pages, int tiles, cudaStream_t stream);

// n_splits CTAs share a row tile's pages (1: none, part unused); part: float32 [n_splits * tiles * 128 * (hd + 2)]
// with tiles = ceil(max_new * nh / nkv / 128) * nkv * B
int wpc_attention_prefill_tc_bounded(const void* q, int q_stride, void* out, int out_stride, const void* k_pages,
                                     const void* v_pages, const int* page_table, int table_width,
                                     const int* cu_seqlens, const int* ctx_lens, int B, int max_new, int nh, int nkv,
                                     int hd, float scale, int window, int sinks, float* lse, int* status, int n_pages,
                                     int n_splits, float* part, cudaStream_t stream);

// Attention with sinks beside a window (sinks > 0, window > 0), or over all earlier positions with what
// the sums of weights need (window = 0, sinks = 0, scores, row_ml / lse given): attention_bounded.cu.
// decode: cluster 0: n_ctas CTAs share all pages (part_o, part_ml, counters as in
// wpc_attention_decode); else `groups` clusters of that size to a pair (as in
// wpc_attention_decode_cluster).  scores: float32 [B * nkv][nh / nkv][score_stride], score_stride a
// multiple of 64 that covers the longest context max_ctx; row_ml: float32 [B][nh][2].  With scores a
// second kernel (wpc_weight_sums_decode, which says what the last arguments are) follows.
int wpc_attention_decode_bounded(const void* q, int q_stride, void* out, int out_stride, const void* k_pages,
                                 const void* v_pages, const int* page_table, int table_width, const int* ctx_lens,
                                 int B, int nh, int nkv, int hd, float scale, int window, int sinks, int n_ctas,
                                 int cluster, int groups, float* part_o, float* part_ml, int* counters, int n_counters,
                                 float* scores, int score_stride, float* row_ml, const int* token_positions, int max_ctx,
                                 int n_pages, float* weight_sums, int* stored_positions, int* status,
                                 cudaStream_t stream);
int wpc_attention_prefill_bounded(const void* q, int q_stride, void* out, int out_stride, const void* k_pages,
                                  const void* v_pages, const int* page_table, int table_width, const int* cu_seqlens,
                                  const int* ctx_lens, int B, int max_new, int nh, int nkv, int hd, float scale,
                                  int window, int sinks, float* lse, int n_pages, cudaStream_t stream);

// attention_sums.cu: the weight that each cached entry received, added to weight_sums
// [n_pages][nkv][64] (an entry of the step's own tokens begins with it, and its place in
// stored_positions gets its token's position).  decode: from what wpc_attention_decode_bounded
// left; plain: from q, k and the rows' log-sums.
int wpc_weight_sums_decode(const float* scores, int score_stride, const float* row_ml, const int* page_table,
                           int table_width, const int* ctx_lens, const int* token_positions, int B, int nh, int nkv,
                           int max_ctx, int n_pages, float* weight_sums, int* stored_positions, int* status,
                           cudaStream_t stream);
int wpc_weight_sums_plain(const void* q, int q_stride, int dtype, const void* k_pages, const int* page_table,
                          int table_width, const int* cu_seqlens, const int* ctx_lens, const int* token_positions,
                          const float* lse, int B, int nh, int nkv, int hd, float scale, int max_new, int max_ctx, int n_pages,
                          float* weight_sums, int* stored_positions, int* status, cudaStream_t stream);

// the same as wpc_weight_sums_plain on the tensor cores (attention_sums_tc.cu): bfloat16, head sizes 64 and 128
int wpc_weight_sums_tc(const void* q, int q_stride, int n_tokens, const void* k_pages, const int* page_table,
                       int table_width, const int* cu_seqlens, const int* ctx_lens, const int* token_positions,
                       const float* lse, int B, int nh, int nkv, int hd, float scale, int max_new, int max_ctx,
                       int n_pages, float* weight_sums, int* stored_positions, int* status, float* part, int* tickets,
                       int n_tickets, cudaStream_t stream);

// the same with mma.sync (attention_sums_mma.cu): bfloat16, head sizes that are multiples of 16 up to 128
int wpc_weight_sums_mma(const void* q, int q_stride, const void* k_pages, const int* page_table, int table_width,
                        const int* cu_seqlens, const int* ctx_lens, const int* token_positions, const float* lse,
                        int B, int nh, int nkv, int hd, float scale, int max_new, int max_ctx, int n_pages,
                        float* weight_sums, int* stored_positions, int* status, cudaStream_t stream);

// eviction.cu.  kept: int32 [layers][B][nkv][keep], the entry that belongs at each place of the kept
// part (-1 behind a shorter sequence).  weight_sums, stored_positions: [layers][n_pages][nkv][64].
int wpc_select_kept(const float* weight_sums, const int* stored_positions, const int* page_table, int table_width,
                    const int* lens, const int* next_positions, int layers, int B, int nkv, int n_pages,
                    int keep, int sinks, int recent, int* kept, int* scratch, int* status, cudaStream_t stream);
// ints of scratch memory that it needs for every (layer, sequence, KV head) (0: scratch may be null)
long wpc_select_kept_scratch(int keep, int table_width);
// k_bytes, v_bytes: bytes of an entry's key and value
int wpc_move_kept(void* k_pages, void* v_pages, int k_bytes, int v_bytes, float* weight_sums, int* stored_positions,
                  const int* page_table, int table_width, const int* kept, int layers, int B, int nkv, int n_pages,
                  int keep, int* status, cudaStream_t stream);

int wpc_sample(const float* logits, int n_rows, int V, const int* slots, long long* seq_state, float temperature,
               const int* banned, int n_banned, int* out, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
