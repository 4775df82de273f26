// The weight that every cached entry received from a step's queries: for entry j of KV head g
//
//   sum[j] = sum over the step's queries t that see j, and the heads h of g's group, of
//            exp(q_th . k_j * scale - max_th) / total_th
//
// the column sums of the attention's softmax, which the choice of the entries that stay in a
// bounded cache goes by (eviction.cu).  They are added to `weight_sums` [page][kv head][place];
// an entry of this step's own tokens has no earlier sum: it begins with this one, and its place in
// `stored_positions` gets the position of its token.  Every sum has one owner that adds in a
// fixed order: no atomics, the same bits every run.
//
//   decode   the attention kernel left its scores and each row's maximum and inverse sum in
//            scratch memory (attention_bounded.cu); a thread to a key adds the group's heads.
//            Bound by the reading of the scores, 4 bytes for each key and head, from L2.
//   prefill  scores once more as matrix products on the tensor cores (attention_sums_tc.cu).
//   plain    any type, head size and number of queries: scores once more from q and k, on the
//            CUDA cores, normalised by the rows' log-sums.
#include "api.h"
#include "attention_sums.cuh"

namespace wpc {

constexpr float SUMS_LOG2E = 1.4426950408889634f;

constexpr int SUMS_THREADS = 256;

__global__ void __launch_bounds__(SUMS_THREADS)
decode_sums_kernel(const float* scores, int score_stride, const float2* row_ml,
                   const int* __restrict__ ctx_lens, int nh, int nkv, SumsTarget t) {
  pdl_trigger();
  pdl_wait();
  const int g = blockIdx.y, b = blockIdx.z, n_rep = nh / nkv;
  const int key = blockIdx.x * SUMS_THREADS + threadIdx.x;
  const int L = ctx_lens[b];
  if (key >= min(L, score_stride)) return;
  const float* s = scores + ((size_t)(b * nkv + g) * n_rep) * score_stride + key;
  const float2* ml = row_ml + (size_t)b * nh + g * n_rep;
  float w = 0.f;
#pragma unroll 8
  for (int r = 0; r < n_rep; ++r) {
    const float2 m = ml[r];
    w += exp2f(s[(size_t)r * score_stride] - m.x) * m.y;
  }
  add_sum(t, nkv, b, g, key, key == L - 1 ? b : -1, w);
}

constexpr int SUMS_ROWS = 16;       // (token, head) rows of q in shared memory at a time

template <typename T>
__global__ void __launch_bounds__(SUMS_THREADS)
sums_plain_kernel(const T* q, int q_stride, const T* k_pages,
                  const int* __restrict__ cu_seqlens, const int* __restrict__ ctx_lens, const float* lse,
                  int nh, int nkv, int hd, float scale, SumsTarget t) {
  pdl_trigger();
  pdl_wait();
  extern __shared__ float smem[];
  float* ks = smem;                               // [PAGE][hd + 1]
  float* qs = ks + WPC_PAGE * (hd + 1);           // [SUMS_ROWS][hd]
  __shared__ float part[4][WPC_PAGE];
  const int blk = blockIdx.x, g = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int n_rep = nh / nkv, L = ctx_lens[b];
  if (blk * WPC_PAGE >= L || blk >= t.table_width) return;
  const int tok0 = cu_seqlens[b], n_new = cu_seqlens[b + 1] - tok0, start = L - n_new;
  const int page = min(max(t.page_table[(size_t)b * t.table_width + blk], 0), t.n_pages - 1);
  const T* kp = k_pages + ((size_t)page * nkv + g) * WPC_PAGE * hd;
  for (int e = tid; e < WPC_PAGE * hd; e += SUMS_THREADS) {
    const int row = e / hd, d = e - row * hd;
    ks[row * (hd + 1) + d] = to_float(kp[e]);
  }
  const int key = blk * WPC_PAGE + (tid & 63), quarter = tid >> 6;
  float w = 0.f;
  const int n_rows = n_new * n_rep;
  for (int r0 = max(blk * WPC_PAGE - start, 0) * n_rep; r0 < n_rows; r0 += SUMS_ROWS) {
    __syncthreads();
    for (int e = tid; e < SUMS_ROWS * hd; e += SUMS_THREADS) {
      const int r = r0 + e / hd, d = e % hd;
      if (r < n_rows) qs[e] = to_float(q[(size_t)(tok0 + r / n_rep) * q_stride + (size_t)(g * n_rep + r % n_rep) * hd + d]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SUMS_ROWS / 4; ++i) {
      const int r = r0 + quarter * (SUMS_ROWS / 4) + i;
      if (r < n_rows && key <= start + r / n_rep) {
        const float* qr = qs + (quarter * (SUMS_ROWS / 4) + i) * hd;
        const float* kr = ks + (tid & 63) * (hd + 1);
        float dot = 0.f;
        for (int d = 0; d < hd; ++d) dot = fmaf(qr[d], kr[d], dot);
        w += exp2f(dot * (scale * SUMS_LOG2E) - lse[(size_t)(tok0 + r / n_rep) * nh + g * n_rep + r % n_rep]);
      }
    }
  }
  part[quarter][tid & 63] = w;
  __syncthreads();
  if (quarter == 0 && key < L) {
    w = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
    add_sum(t, nkv, b, g, key, key >= start ? tok0 + key - start : -1, w);
  }
}

}  // namespace wpc

using namespace wpc;

extern "C" {

int wpc_weight_sums_decode(const float* scores, int score_stride, const float* row_ml, const int* page_table,
                           int table_width, const int* ctx_lens, const int* token_positions, int B, int nh, int nkv,
                           int max_ctx, int n_pages, float* weight_sums, int* stored_positions, int* status,
                           cudaStream_t stream) {
  if (B <= 0 || max_ctx <= 0) return 0;
  if (nkv < 1 || nh % nkv || B > 65535 || nkv > 65535) return WPC_ERR_UNSUPPORTED;
  if (!scores || !row_ml || score_stride < max_ctx || n_pages < 1) return WPC_ERR_BAD_ARGUMENT;
  const SumsTarget t{page_table, table_width, n_pages, token_positions, weight_sums, stored_positions, status};
  wpc::launch(decode_sums_kernel, dim3((max_ctx + SUMS_THREADS - 1) / SUMS_THREADS, nkv, B), SUMS_THREADS, 0, stream,
              scores, score_stride, (const float2*)row_ml, ctx_lens, nh, nkv, t);
  return launch_status();
}

int wpc_weight_sums_plain(const void* q, int q_stride, int dtype, const void* k_pages, const int* page_table,
                          int table_width, const int* cu_seqlens, const int* ctx_lens, const int* token_positions,
                          const float* lse, int B, int nh, int nkv, int hd, float scale, int max_ctx, int n_pages,
                          float* weight_sums, int* stored_positions, int* status, cudaStream_t stream) {
  if (B <= 0 || max_ctx <= 0) return 0;
  if (hd < 1 || hd > 256 || nkv < 1 || nh % nkv || B > 65535 || nkv > 65535) return WPC_ERR_UNSUPPORTED;
  if (!lse || n_pages < 1) return WPC_ERR_BAD_ARGUMENT;
  const SumsTarget t{page_table, table_width, n_pages, token_positions, weight_sums, stored_positions, status};
  const int smem = (WPC_PAGE * (hd + 1) + SUMS_ROWS * hd) * (int)sizeof(float);
  const dim3 grid((max_ctx + WPC_PAGE - 1) / WPC_PAGE, nkv, B);
  WPC_DISPATCH_DTYPE(dtype, Tt, {
    static int configured[MAX_DEVICES];
    if (int rc = allow_smem(sums_plain_kernel<Tt>, smem, configured)) return rc;
    wpc::launch(sums_plain_kernel<Tt>, grid, SUMS_THREADS, smem, stream, (const Tt*)q, q_stride, (const Tt*)k_pages,
                cu_seqlens, ctx_lens, lse, nh, nkv, hd, scale, t);
  });
  return launch_status();
}

}  // extern "C"
