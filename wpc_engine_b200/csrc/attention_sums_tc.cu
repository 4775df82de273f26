// The sums of attention weights (attention_sums.cu) of a prompt's or a chunk's queries, as matrix
// products on the 5th-generation tensor cores:
//
//   sum[j] = sum over queries t and heads h of exp2(q_th . k_j * scale * log2(e) - lse2_th)
//
// with lse2 = maximum + log2(sum) of each row, which the attention kernel left.  The scores are
// computed the other way round, S^T = K Q^T: the 128 keys of two pages are the rows of the MMA, the
// (token, head) rows of the queries its 128 columns, so a key is a lane of tensor memory and one
// thread adds up a key's weights in registers over all queries: no atomics, no scratch memory.
// The CTAs of a cluster share the queries of a key tile, every C-th query tile each, so that
// few keys with many queries fill the device too; rank 0 adds their sums in rank order.
//
// A query tile is as many whole tokens as fit 128 rows (18 of 7 heads): one 3D TMA box of
// [tokens][heads of the group][64] elements for each 64-wide half of a head.  Warps 0..3 add, one
// thread of warp 4 issues the MMAs, one of warp 5 the copies; they meet at mbarriers:
//
//   k_full           TMA -> MMA        the keys have landed
//   q_full[NS]       TMA -> MMA        a query tile has landed
//   q_empty[NS]      MMA -> TMA        the MMAs that read it have finished
//   s_full[2]        MMA -> threads    a tile's scores are in tensor memory
//   s_empty[2]       threads -> MMA    they have been read (128 arrivals)
#include <cuda.h>

#include "api.h"
#include "attention_sums.cuh"
#include "attention_tc.cuh"
#include "common.cuh"
#include "tensor_map.h"

namespace wpc {
namespace fatc {

constexpr int ST_KEYS = 128;             // keys of a CTA: two pages
constexpr int ST_COLS = 128;             // (token, head) rows of a query tile, padded
constexpr int ST_THREADS = 192;
constexpr int ST_MAX_CLUSTER = 8;

template <int HD>
struct StCfg {
  static constexpr int NB = HD / 64;
  static constexpr int STAGES = 4 / NB;                      // query tiles in flight
  static constexpr int HALF = 128 * 128;                     // 128 rows of 64 elements
  static constexpr int TILE = NB * HALF;                     // keys, or one query tile
  static constexpr int SMEM = 1024 + (1 + STAGES) * TILE;
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// A barrier of the 128 adding threads; true if `ok` holds for all of them.
__device__ __forceinline__ bool all_of_128(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 1, 128, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"((uint32_t)ok)
      : "memory");
  return all != 0;
}

template <int HD>
__global__ void __launch_bounds__(ST_THREADS, 2)
prefill_sums_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_q,
                    const int* __restrict__ cu_seqlens, const int* __restrict__ ctx_lens, const float* lse,
                    int nh, int nkv, int C, int tile_tokens, float scale_log2, const SumsTarget t,
                    unsigned long long wait_ns, int starve, int late_trigger) {
  using W = StCfg<HD>;
  constexpr int ST_STAGES = W::STAGES;
  pdl_wait();
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ __align__(16) float s_lse[2][ST_COLS];          // minus the columns' log-sums, -inf where there is no row
  __shared__ __align__(16) int s_pos[2][ST_COLS];            // places of the columns' queries, -1 where there is no row
  __shared__ float s_part[ST_MAX_CLUSTER][ST_KEYS];          // rank 0: the ranks' sums
  __shared__ __align__(8) uint64_t bars[1 + 2 * ST_STAGES + 4];
  __shared__ uint32_t tmem_holder;
  __shared__ int failed;
  uint64_t *k_full = bars, *q_full = bars + 1, *q_empty = q_full + ST_STAGES, *s_full = q_empty + ST_STAGES, *s_empty = s_full + 2;
  const int rank = blockIdx.x % C, g = blockIdx.x / C, kt = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n_rep = nh / nkv;
  const int L = ctx_lens[b], tok0 = cu_seqlens[b], n_new = cu_seqlens[b + 1] - tok0, start = L - n_new;
  const int key0 = kt * ST_KEYS;
  if (key0 >= L || n_new <= 0) return;                       // the whole cluster, before any barrier
  const int t_first = max(0, key0 - start);                  // the first token that sees a key of the tile
  const int n_tiles = (n_new - t_first + tile_tokens - 1) / tile_tokens;
  const int mine = n_tiles > rank ? (n_tiles - rank + C - 1) / C : 0;   // tiles rank, rank + C, ..
  if (C > 1) cluster_arrive();

  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t k_s = smem_u32(base), q_s = k_s + W::TILE;
  const int rows = n_rep * tile_tokens;
  if (tid == 0) {
    mbar_init(k_full, 1);
    for (int i = 0; i < ST_STAGES; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(s_empty + i, 128);
    }
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // columns behind the last row of a query tile are never copied: zeros, so that their scores are finite
  for (int e = tid; e < ST_STAGES * W::NB * (ST_COLS - rows) * 8; e += ST_THREADS) {
    const int half = e / ((ST_COLS - rows) * 8), in = e - half * ((ST_COLS - rows) * 8);
    *(uint4*)(base + W::TILE + half * W::HALF + rows * 128 + in * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_async_smem();
  if (warp == 4) tmem_alloc(&tmem_holder, 256);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_holder;
  // (only now: the kernel behind may hold tensor memory while it waits for this one, so every CTA
  // of this one must have got its own first)
  if (!late_trigger) pdl_trigger();
  float w = 0.f;

  if (warp == 5) {
    if (lane == 0 && !starve) {
      const int* table = t.page_table + (size_t)b * t.table_width;
      if (mine) {
        mbar_expect_tx(k_full, W::TILE);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int block = key0 / WPC_PAGE + p;
          const int page = block * WPC_PAGE < L && block < t.table_width ? min(max(table[block], 0), t.n_pages - 1) : 0;
#pragma unroll
          for (int hb = 0; hb < W::NB; ++hb)
            tma_load_2d(k_s + hb * W::HALF + p * (WPC_PAGE * 128), &map_k, hb * 64, (page * nkv + g) * WPC_PAGE, k_full);
        }
      }
      for (int i = 0; i < mine; ++i) {
        const int st = i % ST_STAGES;
        if (!mbar_wait(q_empty + st, ((i / ST_STAGES) & 1) ^ 1, wait_ns)) { atomicExch(&failed, 1); break; }
        mbar_expect_tx(q_full + st, rows * 128 * W::NB);
#pragma unroll
        for (int hb = 0; hb < W::NB; ++hb)
          tma_load_3d(q_s + st * W::TILE + hb * W::HALF, &map_q, hb * 64, g * n_rep,
                      tok0 + t_first + (rank + i * C) * tile_tokens, q_full + st);
      }
    }
    if (late_trigger) pdl_trigger();
  } else if (warp == 4) {
    if (lane == 0 && mine) {
      constexpr uint32_t idesc = instr_desc(ST_COLS, false);
      bool ok = mbar_wait(k_full, 0, wait_ns);
      for (int i = 0; ok && i < mine; ++i) {
        const int st = i % ST_STAGES;
        ok = mbar_wait(q_full + st, (i / ST_STAGES) & 1, wait_ns) && mbar_wait(s_empty + (i & 1), ((i >> 1) & 1) ^ 1, wait_ns);
        if (!ok) break;
        fence_after_sync();
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t off = (kk >> 2) * W::HALF + (kk & 3) * 32;
          umma_bf16(tmem + (i & 1) * ST_COLS, smem_desc(k_s + off, 16), smem_desc(q_s + st * W::TILE + off, 16), idesc,
                    kk > 0 ? 1u : 0u);
        }
        umma_commit(s_full + (i & 1));
        umma_commit(q_empty + st);
      }
      if (!ok) atomicExch(&failed, 1);
    }
  } else {
    // ---- thread r owns key key0 + r ----
    const int key = key0 + tid;
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    const int my_tok = tid / n_rep, my_head = g * n_rep + tid % n_rep;
    auto token_of = [&](int i) { return t_first + (rank + i * C) * tile_tokens + my_tok; };
    auto lse_of = [&](int i) {
      const int tok = token_of(i);
      return i < mine && tid < rows && tok < n_new ? -lse[(size_t)(tok0 + tok) * nh + my_head] : -INFINITY;
    };
    float next_lse = lse_of(0);
    float2 acc[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    const float2 scale2 = make_float2(scale_log2, scale_log2);
    bool ok = true;
    for (int i = 0; i < mine; ++i) {
      const int bb = i & 1, tile_first = t_first + (rank + i * C) * tile_tokens;
      // keys that not every query sees, or columns that are no rows of this sequence
      const bool masked = key0 + ST_KEYS - 1 > start + tile_first || tile_first + tile_tokens > n_new;
      s_lse[bb][tid] = next_lse;
      if (masked) s_pos[bb][tid] = tid < rows && token_of(i) < n_new ? start + token_of(i) : -1;
      next_lse = lse_of(i + 1);
      if (!all_of_128(ok)) break;                            // (a wait of the tile before ran out for some warp)
      ok = mbar_wait(s_full + bb, (i >> 1) & 1, wait_ns);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) continue;
      fence_after_sync();
#pragma unroll
      for (int c = 0; c < ST_COLS; c += 32) {
        uint32_t su[32];
        tmem_ld32(tmem + bb * ST_COLS + lane_off + c, su);
        tmem_ld_wait();
        if (c == ST_COLS - 32) {
          fence_before_sync();
          mbar_arrive(s_empty + bb);
        }
        if (masked) {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float x = fmaf(__uint_as_float(su[j]), scale_log2, s_lse[bb][c + j]);
            const float p = key <= s_pos[bb][c + j] ? ex2(x) : 0.f;
            if (j & 1) acc[(j >> 1) & 3].y += p; else acc[(j >> 1) & 3].x += p;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 l = *(const float4*)&s_lse[bb][c + j];
            const float2 x0 = __ffma2_rn(make_float2(__uint_as_float(su[j]), __uint_as_float(su[j + 1])), scale2, make_float2(l.x, l.y));
            const float2 x1 = __ffma2_rn(make_float2(__uint_as_float(su[j + 2]), __uint_as_float(su[j + 3])), scale2, make_float2(l.z, l.w));
            acc[(j >> 1) & 3] = __fadd2_rn(acc[(j >> 1) & 3], make_float2(ex2(x0.x), ex2(x0.y)));
            acc[((j >> 1) + 1) & 3] = __fadd2_rn(acc[((j >> 1) + 1) & 3], make_float2(ex2(x1.x), ex2(x1.y)));
          }
        }
      }
    }
    if (!ok) atomicExch(&failed, 1);
    w = ((acc[0].x + acc[0].y) + (acc[1].x + acc[1].y)) + ((acc[2].x + acc[2].y) + (acc[3].x + acc[3].y));
  }
  fence_before_sync();
  __syncthreads();
  if (failed) {
    // a wait ran out: give copies and MMAs in flight time to land
    if (tid == 0 && t.status) atomicExch(t.status, WPC_ERR_DEVICE_WAIT);
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  // tensor memory goes back before anything waits for the other ranks: a CTA that waits for room
  // in it, here or in another kernel, never waits for one that waits in turn
  if (warp == 4) {
    fence_after_sync();
    tmem_dealloc(tmem, 256);
  }
  if (C > 1) {
    cluster_wait();                                          // (every rank has begun: rank 0's memory may be written)
    if (tid < ST_KEYS) {
      const uint32_t to = peer_smem(smem_u32(&s_part[rank][tid]), 0u);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(w) : "memory");
    }
    cluster_arrive();
    cluster_wait();
    if (rank == 0 && tid < ST_KEYS) {
      w = s_part[0][tid];
      for (int r = 1; r < C; ++r) w += s_part[r][tid];
    }
  }
  if (rank == 0 && tid < ST_KEYS && key0 + tid < L) {
    const int key = key0 + tid;
    add_sum(t, nkv, b, g, key, key >= start ? tok0 + key - start : -1, w);
  }
}

template <int HD>
static int launch_sums(const void* q, int q_stride, int n_tokens, const void* k_pages, const int* cu_seqlens,
                       const int* ctx_lens, const float* lse, int B, int nh, int nkv, float scale, int max_new,
                       int max_ctx, const SumsTarget& t, cudaStream_t stream) {
  static int configured[MAX_DEVICES];
  if (int rc = allow_smem(prefill_sums_kernel<HD>, StCfg<HD>::SMEM, configured)) return rc;
  const int n_rep = nh / nkv, tile_tokens = ST_COLS / n_rep;
  const long cache_rows = (long)t.n_pages * nkv * WPC_PAGE;
  if (cache_rows > 0x7fffffffL) return WPC_ERR_TOO_LARGE;
  CUtensorMap mk, mq;
  if (int rc = tc::tensor_map(k_pages, (int)cache_rows, HD, HD, WPC_PAGE, &mk)) return rc;
  if (int rc = tc::tensor_map_heads(q, n_tokens, nh, HD, q_stride, tile_tokens, n_rep, &mq)) return rc;
  // as many CTAs to a key tile as leave every SM two to begin with and each at least two query tiles
  const int key_tiles = (max_ctx + ST_KEYS - 1) / ST_KEYS;
  const long tiles = (long)key_tiles * nkv * B, query_tiles = (max_new + tile_tokens - 1) / tile_tokens;
  int C = 1;
  while (C < ST_MAX_CLUSTER && tiles * C < 4L * sm_count() && query_tiles >= 4L * C) C *= 2;
  if (key_tiles > 65535 || B > 65535) return WPC_ERR_TOO_LARGE;
  wpc::launch_clusters(prefill_sums_kernel<HD>, dim3((unsigned)(C * nkv), (unsigned)key_tiles, (unsigned)B), ST_THREADS,
                       StCfg<HD>::SMEM, stream, (unsigned)C, mk, mq, cu_seqlens, ctx_lens, lse, nh, nkv, C, tile_tokens,
                       scale * 1.4426950408889634f, t, wait_policy().limit_ns, wait_policy().starve, max_new >= 1024 ? 1 : 0);
  return launch_status();
}

}  // namespace fatc
}  // namespace wpc

extern "C" {

// Head sizes 64 and 128, at most 128 heads to a group; q rows 16-byte aligned (q_stride a multiple of 8).
int wpc_weight_sums_tc(const void* q, int q_stride, int n_tokens, const void* k_pages, const int* page_table,
                       int table_width, const int* cu_seqlens, const int* ctx_lens, const int* token_positions,
                       const float* lse, int B, int nh, int nkv, int hd, float scale, int max_new, int max_ctx,
                       int n_pages, float* weight_sums, int* stored_positions, int* status, cudaStream_t stream) {
  if (B <= 0 || max_new <= 0 || max_ctx <= 0) return 0;
  if (!wpc_attention_prefill_tc_supports(nh, nkv, hd) || q_stride % 8 || (((uintptr_t)q | (uintptr_t)k_pages) & 15))
    return WPC_ERR_UNSUPPORTED;
  if (!lse || n_pages < 1) return WPC_ERR_BAD_ARGUMENT;
  const wpc::SumsTarget t{page_table, table_width, n_pages, token_positions, weight_sums, stored_positions, status};
  if (hd == 128)
    return wpc::fatc::launch_sums<128>(q, q_stride, n_tokens, k_pages, cu_seqlens, ctx_lens, lse, B, nh, nkv, scale,
                                       max_new, max_ctx, t, stream);
  return wpc::fatc::launch_sums<64>(q, q_stride, n_tokens, k_pages, cu_seqlens, ctx_lens, lse, B, nh, nkv, scale,
                                    max_new, max_ctx, t, stream);
}

}  // extern "C"
