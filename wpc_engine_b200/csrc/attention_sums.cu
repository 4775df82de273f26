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
//            Bound by the reading of the scores, 4 bytes for each key and head, from L2: 2 us beside
//            the attention at 8 sequences of 4,001 (28 heads).
//   prefill  scores once more as matrix products on the tensor cores (attention_sums_tc.cu,
//            attention_sums_mma.cu), normalised by the rows' log-sums.
//   plain    the same on the CUDA cores, for any type, head size and alignment: the 32-bit path's.
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
  const int stated = ctx_lens[b], L = min(stated, t.table_width * WPC_PAGE);
  if (key == 0 && g == 0) check_length(t, stated, score_stride);
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

// The plain kernel: a CTA takes a page of keys of one KV head, its four groups of 64 threads (a thread to a
// key) eight (token, head) rows of the queries each at a time, all from shared memory as float32.  With
// few keys and many queries the CTAs of a cluster share the queries, every C-th tile each, and rank 0
// adds their sums in rank order.  160 queries of 14 heads of 64 over 400 keys, two sequences: 841 us with
// four rows, one element a load and no clusters, 203 us this way (attention included).  Copies to shared memory
// one load and store at a time instead of in groups: 85.6 against 80.5 us, 200 tokens over themselves.
constexpr int SUMS_ROWS = 32;       // (token, head) rows of q in shared memory at a time
constexpr int SUMS_MAX_CLUSTER = 8;
constexpr int SUMS_COPY = 8;        // elements that a thread copies at a time

// VEC: head_dim is a multiple of four, so that rows are read four elements a load (rows of hd + 4
// floats keep the threads of a quarter-warp on different banks; rows of hd + 1 do so one by one).
template <typename T, bool VEC>
__global__ void __launch_bounds__(SUMS_THREADS)
sums_plain_kernel(const T* q, int q_stride, const T* k_pages, const int* __restrict__ cu_seqlens,
                  const int* __restrict__ ctx_lens, const float* lse, int nh, int nkv, int hd, int C, float scale_log2,
                  SumsTarget t) {
  pdl_trigger();
  pdl_wait();
  extern __shared__ __align__(16) float smem[];
  const int k_stride = VEC ? hd + 4 : hd + 1;
  float* ks = smem;                               // [PAGE][k_stride]
  float* qs = ks + WPC_PAGE * k_stride;           // [SUMS_ROWS][hd]
  __shared__ float s_group[4][WPC_PAGE], s_part[SUMS_MAX_CLUSTER][WPC_PAGE];
  const int rank = blockIdx.x % C, blk = blockIdx.x / C, g = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int n_rep = nh / nkv, L = min(ctx_lens[b], t.table_width * WPC_PAGE);
  const int tok0 = cu_seqlens[b], n_new = cu_seqlens[b + 1] - tok0, start = L - n_new;
  if (blk == 0 && rank == 0 && g == 0 && tid == 0) check_length(t, ctx_lens[b], (int)(gridDim.x / C) * WPC_PAGE);
  if (blk * WPC_PAGE >= L || blk >= t.table_width) return;       // the whole cluster, before any barrier
  if (C > 1) cluster_arrive();
  const int page = min(max(t.page_table[(size_t)b * t.table_width + blk], 0), t.n_pages - 1);
  const T* kp = k_pages + ((size_t)page * nkv + g) * WPC_PAGE * hd;
  // (loads in groups ahead of their stores, which they cannot be moved across)
  if (VEC) {
    for (int e0 = tid * 4; e0 < WPC_PAGE * hd; e0 += 16 * SUMS_THREADS) {
      float4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (e0 + u * 4 * SUMS_THREADS < WPC_PAGE * hd) v[u] = load4(kp + e0 + u * 4 * SUMS_THREADS);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int e = e0 + u * 4 * SUMS_THREADS, row = e / hd;
        if (e < WPC_PAGE * hd) *(float4*)(ks + row * k_stride + e - row * hd) = v[u];
      }
    }
  } else {
    for (int e = tid; e < WPC_PAGE * hd; e += SUMS_THREADS) {
      const int row = e / hd, d = e - row * hd;
      ks[row * k_stride + d] = to_float(kp[e]);
    }
  }
  const int place = tid & 63, key = blk * WPC_PAGE + place, group = tid >> 6;
  const float* kr = ks + place * k_stride;
  float w = 0.f;
  const int n_rows = n_new * n_rep;
  for (int r0 = max(blk * WPC_PAGE - start, 0) * n_rep + rank * SUMS_ROWS; r0 < n_rows; r0 += C * SUMS_ROWS) {
    __syncthreads();
    for (int e0 = tid; e0 < SUMS_ROWS * hd; e0 += SUMS_COPY * SUMS_THREADS) {
      float v[SUMS_COPY];
#pragma unroll
      for (int u = 0; u < SUMS_COPY; ++u) {
        const int e = e0 + u * SUMS_THREADS, r = r0 + e / hd, d = e % hd;
        v[u] = e < SUMS_ROWS * hd && r < n_rows
                   ? to_float(q[(size_t)(tok0 + r / n_rep) * q_stride + (size_t)(g * n_rep + r % n_rep) * hd + d]) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < SUMS_COPY; ++u)
        if (e0 + u * SUMS_THREADS < SUMS_ROWS * hd) qs[e0 + u * SUMS_THREADS] = v[u];
    }
    __syncthreads();
    // group `group` takes rows group, group + 4, ..
    const float* qr = qs + group * hd;
    const int rows = (min(n_rows - r0, SUMS_ROWS) - group + 3) / 4;
    float dot[SUMS_ROWS / 4];
#pragma unroll
    for (int i = 0; i < SUMS_ROWS / 4; ++i) dot[i] = 0.f;
    if (rows <= 2) {                              // (the few rows of a single token)
      for (int i = 0; i < rows; ++i) {
        const float* q0 = qr + i * 4 * hd;
        float d0 = 0.f;
        if (VEC) {
          for (int d = 0; d < hd; d += 4) {
            const float4 k4 = *(const float4*)(kr + d), q4 = *(const float4*)(q0 + d);
            d0 = fmaf(q4.x, k4.x, d0);
            d0 = fmaf(q4.y, k4.y, d0);
            d0 = fmaf(q4.z, k4.z, d0);
            d0 = fmaf(q4.w, k4.w, d0);
          }
        } else {
          for (int d = 0; d < hd; ++d) d0 = fmaf(q0[d], kr[d], d0);
        }
        if (i == 0) dot[0] = d0;
        else dot[1] = d0;
      }
    } else if (VEC) {
      for (int d = 0; d < hd; d += 4) {
        const float4 k4 = *(const float4*)(kr + d);
#pragma unroll
        for (int i = 0; i < SUMS_ROWS / 4; ++i) {
          const float4 q4 = *(const float4*)(qr + i * 4 * hd + d);
          dot[i] = fmaf(q4.x, k4.x, dot[i]);
          dot[i] = fmaf(q4.y, k4.y, dot[i]);
          dot[i] = fmaf(q4.z, k4.z, dot[i]);
          dot[i] = fmaf(q4.w, k4.w, dot[i]);
        }
      }
    } else {
      for (int d = 0; d < hd; ++d)
#pragma unroll
        for (int i = 0; i < SUMS_ROWS / 4; ++i) dot[i] = fmaf(qr[i * 4 * hd + d], kr[d], dot[i]);
    }
#pragma unroll
    for (int i = 0; i < SUMS_ROWS / 4; ++i) {
      const int r = r0 + i * 4 + group;
      if (i < rows && key <= start + r / n_rep)
        w += exp2f(dot[i] * scale_log2 - lse[(size_t)(tok0 + r / n_rep) * nh + g * n_rep + r % n_rep]);
    }
  }
  s_group[group][place] = w;
  __syncthreads();
  if (C > 1) cluster_wait();                      // (every rank has begun: rank 0's memory may be written)
  if (group == 0) {
    w = (s_group[0][place] + s_group[1][place]) + (s_group[2][place] + s_group[3][place]);
    if (C > 1) {
      const uint32_t to = peer_smem((uint32_t)__cvta_generic_to_shared(&s_part[rank][place]), 0u);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(w) : "memory");
    }
  }
  if (C > 1) {
    cluster_arrive();
    cluster_wait();
    w = 0.f;
    if (rank == 0)
      for (int c = 0; c < C; ++c) w += s_part[c][place];
  }
  if (rank == 0 && group == 0 && key < L) add_sum(t, nkv, b, g, key, key >= start ? tok0 + key - start : -1, w);
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
                          const float* lse, int B, int nh, int nkv, int hd, float scale, int max_new, int max_ctx,
                          int n_pages, float* weight_sums, int* stored_positions, int* status, cudaStream_t stream) {
  if (B <= 0 || max_ctx <= 0) return 0;
  if (hd < 1 || hd > 256 || nkv < 1 || nh % nkv || B > 65535 || nkv > 65535) return WPC_ERR_UNSUPPORTED;
  if (!lse || n_pages < 1 || max_new < 1) return WPC_ERR_BAD_ARGUMENT;
  const SumsTarget t{page_table, table_width, n_pages, token_positions, weight_sums, stored_positions, status};
  const bool vec = hd % 4 == 0 && (uintptr_t)k_pages % 16 == 0;
  const int smem = (WPC_PAGE * (vec ? hd + 4 : hd + 1) + SUMS_ROWS * hd) * (int)sizeof(float);
  // as many CTAs to a page as give every SM two, each at least two tiles
  const int pages = (max_ctx + WPC_PAGE - 1) / WPC_PAGE;
  const long tiles = ((long)max_new * (nh / nkv) + SUMS_ROWS - 1) / SUMS_ROWS;
  int C = 1;
  while (C < SUMS_MAX_CLUSTER && (long)pages * nkv * B * C < 2L * sm_count() && tiles >= 4L * C) C *= 2;
  const dim3 grid((unsigned)(pages * C), nkv, B);
  auto go = [&](auto kernel, auto* q_, auto* k_, int (&configured)[MAX_DEVICES]) {
    if (int rc = allow_smem(kernel, smem, configured)) return rc;
    wpc::launch_clusters(kernel, grid, SUMS_THREADS, smem, stream, (unsigned)C, q_, q_stride, k_, cu_seqlens, ctx_lens, lse, nh,
                         nkv, hd, C, scale * SUMS_LOG2E, t);
    return launch_status();
  };
  WPC_DISPATCH_DTYPE(dtype, Tt, {
    static int with_vec[MAX_DEVICES], without[MAX_DEVICES];
    return vec ? go(sums_plain_kernel<Tt, true>, (const Tt*)q, (const Tt*)k_pages, with_vec)
               : go(sums_plain_kernel<Tt, false>, (const Tt*)q, (const Tt*)k_pages, without);
  });
  return WPC_ERR_BAD_ARGUMENT;
}

}  // extern "C"
