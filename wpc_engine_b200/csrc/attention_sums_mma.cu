// The sums of attention weights (attention_sums.cu) of several queries a sequence with mma.sync, for the
// bfloat16 head sizes that attention_sums_tc.cu does not take (multiples of 16 up to 128):
//
//   sum[j] = sum over queries t and heads h of exp2(q_th . k_j * scale * log2(e) - lse2_th)
//
// A CTA takes a page of keys of one KV head; its four warps hold 16 keys each as the MMA's rows, in
// registers for the whole kernel, and 64 (token, head) rows of the queries at a time are the
// columns, copied to shared memory one tile ahead.  A thread adds the weights of two keys, the
// four threads that share them add up at the end.  With few keys and many queries the CTAs of a
// cluster share the queries, every C-th tile each, and rank 0 adds their sums in rank order: the
// same bits every run.  1,000 queries of 4 heads of 48 (2 KV heads) over themselves take 28 us with
// the attention, 18 of them without sums; 2,048 behind 3,952 earlier positions 201, 102 of them without.
// Alone this kernel takes 47 there, no unit full (exponentials 36 %, matrix pipe 19 %; the warps wait for fixed
// latencies, shared memory and the barriers around a tile); behind the attention its CTAs become
// resident early, crowded on the SMs that the attention leaves free, and take twice as long (136 in all
// without early starts anywhere).
#include "attention_mma.cuh"
#include "attention_sums.cuh"

namespace wpc {
namespace fa {

constexpr int SM_ROWS = 64;               // query rows a tile
constexpr int SM_MAX_CLUSTER = 8;

template <int HD>
struct SmCfg {
  static constexpr int TILE = SM_ROWS * Cfg<HD>::STRIDE;       // elements
  static constexpr int SMEM = 3 * TILE * 2;                    // the keys, two query tiles
};

template <int HD>
__global__ void __launch_bounds__(THREADS)
sums_mma_kernel(const __nv_bfloat16* q, int q_stride, const __nv_bfloat16* k_pages, const int* __restrict__ cu_seqlens,
                const int* __restrict__ ctx_lens, const float* lse, int nh, int nkv, int C, float scale_log2,
                const SumsTarget t) {
  pdl_trigger();
  pdl_wait();
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __nv_bfloat16* ks = (__nv_bfloat16*)smem_raw;
  __nv_bfloat16* qs = ks + SmCfg<HD>::TILE;                    // [2]
  __shared__ float s_lse[2][SM_ROWS];
  __shared__ int s_pos[2][SM_ROWS];
  __shared__ float s_part[SM_MAX_CLUSTER][PAGE];
  const int rank = blockIdx.x % C, blk = blockIdx.x / C, g = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n_rep = nh / nkv, L = min(ctx_lens[b], t.table_width * WPC_PAGE), tok0 = cu_seqlens[b], n_new = cu_seqlens[b + 1] - tok0, start = L - n_new;
  if (blk == 0 && rank == 0 && g == 0 && tid == 0) check_length(t, ctx_lens[b], (int)(gridDim.x / C) * PAGE);
  if (blk * PAGE >= L || blk >= t.table_width || n_new <= 0) return;      // the whole cluster, before any barrier
  if (C > 1) cluster_arrive();
  const int page = min(max(t.page_table[(size_t)b * t.table_width + blk], 0), t.n_pages - 1);
  load_page<HD>(ks, k_pages + ((size_t)page * nkv + g) * PAGE * HD, tid);
  const int r_first = max(blk * PAGE - start, 0) * n_rep, n_rows = n_new * n_rep;
  const int tiles = (n_rows - r_first + SM_ROWS - 1) / SM_ROWS;
  auto load_queries = [&](int i, int buf) {
    __nv_bfloat16* dst = qs + buf * SmCfg<HD>::TILE;
    constexpr int CPR = HD / 8;
    for (int c = tid; c < SM_ROWS * CPR; c += THREADS) {
      const int row = c / CPR, col = c - row * CPR, r = r_first + i * SM_ROWS + row;
      __nv_bfloat16* to = dst + row * Cfg<HD>::STRIDE + col * 8;
      if (r < n_rows) cp_async16(to, q + (size_t)(tok0 + r / n_rep) * q_stride + (size_t)(g * n_rep + r % n_rep) * HD + col * 8);
      else *(uint4*)to = make_uint4(0, 0, 0, 0);               // (finite scores, which nobody sees)
    }
    if (tid < SM_ROWS) {
      const int r = r_first + i * SM_ROWS + tid;
      s_lse[buf][tid] = r < n_rows ? lse[(size_t)(tok0 + r / n_rep) * nh + g * n_rep + r % n_rep] : 0.f;
      s_pos[buf][tid] = r < n_rows ? start + r / n_rep : -1;
    }
  };
  if (rank < tiles) load_queries(rank, 0);
  cp_async_commit();
  uint32_t kf[HD / 16][4];                                     // this warp's 16 keys as the MMA's A operand
  const int key0 = blk * PAGE + warp * 16 + (lane >> 2);       // the thread's keys: key0 and key0 + 8
  float acc[2] = {0.f, 0.f};
  int n = 0;
  for (int i = rank; i < tiles; i += C, ++n) {
    if (i + C < tiles) load_queries(i + C, (n + 1) & 1);
    cp_async_commit();
    cp_async_wait<1>();
    __syncthreads();
    if (n == 0) {
      const int mat = lane >> 3, r = lane & 7;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
        ldmatrix_x4(kf[kk], ks + (warp * 16 + (mat & 1) * 8 + r) * Cfg<HD>::STRIDE + kk * 16 + (mat >> 1) * 8);
    }
    float s[8][4];
    scores<HD, 8>(kf, qs + (n & 1) * SmCfg<HD>::TILE, 0, s, lane);
#pragma unroll
    for (int nt = 0; nt < 8; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int col = nt * 8 + (lane & 3) * 2 + j;
        const float l = s_lse[n & 1][col];
        const int p = s_pos[n & 1][col];
        acc[0] += key0 <= p ? ex2_fast(fmaf(s[nt][j], scale_log2, -l)) : 0.f;
        acc[1] += key0 + 8 <= p ? ex2_fast(fmaf(s[nt][2 + j], scale_log2, -l)) : 0.f;
      }
    __syncthreads();                                           // the buffer is loaded again
  }
  cp_async_wait<0>();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    acc[h] += __shfl_xor_sync(0xffffffffu, acc[h], 1);
    acc[h] += __shfl_xor_sync(0xffffffffu, acc[h], 2);
  }
  if (C > 1) cluster_wait();                                   // (every rank has begun: rank 0's memory may be written)
  if ((lane & 3) == 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float* part = &s_part[rank][warp * 16 + (lane >> 2) + 8 * h];
      if (C > 1) {
        const uint32_t to = peer_smem(smem_u32(part), 0u);
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(acc[h]) : "memory");
      } else {
        *part = acc[h];
      }
    }
  }
  if (C > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  const int key = blk * PAGE + tid;
  if (rank == 0 && tid < PAGE && key < L) {
    float w = 0.f;
    for (int c = 0; c < C; ++c) w += s_part[c][tid];
    add_sum(t, nkv, b, g, key, key >= start ? tok0 + key - start : -1, w);
  }
}

template <int HD>
static int launch_sums_mma(const void* q, int q_stride, const void* k_pages, const int* cu_seqlens, const int* ctx_lens,
                           const float* lse, int B, int nh, int nkv, float scale, int max_new, int max_ctx,
                           const SumsTarget& t, cudaStream_t stream) {
  static int configured[MAX_DEVICES];
  if (int rc = allow_smem(sums_mma_kernel<HD>, SmCfg<HD>::SMEM, configured)) return rc;
  // as many CTAs to a page as give every SM four, each at least two tiles
  const int pages = (max_ctx + PAGE - 1) / PAGE;
  const long tiles = ((long)max_new * (nh / nkv) + SM_ROWS - 1) / SM_ROWS;
  int C = 1;
  while (C < SM_MAX_CLUSTER && (long)pages * nkv * B * C < 4L * sm_count() && tiles >= 4L * C) C *= 2;
  wpc::launch_clusters(sums_mma_kernel<HD>, dim3((unsigned)(pages * C), (unsigned)nkv, (unsigned)B), THREADS, SmCfg<HD>::SMEM,
                       stream, (unsigned)C, (const __nv_bfloat16*)q, q_stride, (const __nv_bfloat16*)k_pages, cu_seqlens,
                       ctx_lens, lse, nh, nkv, C, scale * LOG2E, t);
  return launch_status();
}

}  // namespace fa
}  // namespace wpc

using namespace wpc;

extern "C" int wpc_weight_sums_mma(const void* q, int q_stride, const void* k_pages, const int* page_table, int table_width,
                                   const int* cu_seqlens, const int* ctx_lens, const int* token_positions, const float* lse,
                                   int B, int nh, int nkv, int hd, float scale, int max_new, int max_ctx, int n_pages,
                                   float* weight_sums, int* stored_positions, int* status, cudaStream_t stream) {
  if (B <= 0 || max_new <= 0 || max_ctx <= 0) return 0;
  if (!wpc_attention_mma_supports(nh, nkv, hd) || q_stride % 8 || (((uintptr_t)q | (uintptr_t)k_pages) & 15) || B > 65535 ||
      nkv > 65535)
    return WPC_ERR_UNSUPPORTED;
  if (!lse || n_pages < 1) return WPC_ERR_BAD_ARGUMENT;
  const SumsTarget t{page_table, table_width, n_pages, token_positions, weight_sums, stored_positions, status};
  WPC_DISPATCH_HD(hd, fa::launch_sums_mma<HD>(q, q_stride, k_pages, cu_seqlens, ctx_lens, lse, B, nh, nkv, scale, max_new,
                                             max_ctx, t, stream));
}
