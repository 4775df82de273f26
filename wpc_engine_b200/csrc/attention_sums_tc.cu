// The sums of attention weights (attention_sums.cu) of a prompt's or a chunk's queries, as matrix
// products on the 5th-generation tensor cores:
//
//   sum[j] = sum over queries t and heads h of exp2(q_th . k_j * scale * log2(e) - lse2_th)
//
// with lse2 = maximum + log2(sum) of each row, which the attention kernel left.  The scores are
// computed the other way round, S^T = K Q^T: the 256 keys of four pages are the rows of two MMAs, the
// (token, head) rows of the queries their 128 columns, so a key is a lane of tensor memory and one
// thread adds up a key's weights in registers over all queries: no atomics on sums.
//
// The work is the list of (sequence, key tile, KV head, query tile) units that have something to see,
// in that order.  One CTA to an SM takes an equal share of the list and walks it as segments of one
// (sequence, key tile, KV head) each, so that every SM does the same number of exponentials,
// whatever the lengths.  A segment that holds all query tiles of its keys adds their sums itself; the
// others leave theirs in scratch memory, and the CTA that takes the keys' last ticket adds them
// in the order of the list (the same bits every run; nobody waits).  A CTA whose wait ran out still takes the
// tickets of all its segments, with a mark, so that they are zero again for the next launch; marked keys
// get no sum.
//
// A query tile is as many whole tokens as fit 128 rows (18 of 7 heads): one 3D TMA box of
// [tokens][heads of the group][64] elements for each 64-wide half of a head.  Warps 0..7 add (four for
// each half of the keys), one thread of warp 8 issues the MMAs, one of warp 9 the copies; they meet
// at mbarriers:
//
//   k_full[2], k_empty[2]     TMA <-> MMA        the keys of a segment (the next one's come early)
//   q_full[NS], q_empty[NS]   TMA <-> MMA        query tiles
//   s_full[2][2]              MMA -> threads     a half's scores of a unit are in tensor memory
//   s_empty[2][2]             threads -> MMA     they have been read (128 arrivals)
//
// Bound by the exponentials: a prompt of 2,048 tokens of the 7B shape (28 heads, 4 KV heads of 128) has 59
// million, 15.7 us at the unit's rate of 16 a cycle and SM; the kernel takes 26 of the call's 69 us, of
// which 8 are the start, the first keys and the tickets (30 of 76 with the copies started after tensor
// memory was there).  A CTA to a key tile, with the queries shared in clusters, instead of equal shares of the list:
// 42.  An eighth or three of the exponentials by a polynomial changed nothing (76.4 and 75.4).
#include <cuda.h>

#include "api.h"
#include "attention_sums.cuh"
#include "attention_tc.cuh"
#include "common.cuh"
#include "tensor_map.h"

namespace wpc {
namespace fatc {

constexpr int ST_KEYS = 256;             // keys of a segment: four pages
constexpr int ST_COLS = 128;             // (token, head) rows of a query tile, padded
constexpr int ST_THREADS = 320;
constexpr int ST_MMA_WARP = 8, ST_COPY_WARP = 9;
constexpr int ST_FAILED = 1 << 16;       // in a ticket: a CTA's wait ran out (the count below it: at most the CTAs of a grid)

template <int HD>
struct StCfg {
  static constexpr int NB = HD / 64;
  static constexpr int STAGES = NB == 2 ? 2 : 6;             // query tiles in flight
  static constexpr int K_HALF = ST_KEYS * 128;               // 256 rows of 64 elements
  static constexpr int K_BYTES = NB * K_HALF;
  static constexpr int Q_HALF = ST_COLS * 128;
  static constexpr int Q_BYTES = NB * Q_HALF;
  static constexpr int SMEM = 1024 + 2 * K_BYTES + STAGES * Q_BYTES;
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// A barrier of `n` threads under number `id`; true if `ok` holds for all of them.
__device__ __forceinline__ bool all_of(int id, int n, bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, %2, %3, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"((uint32_t)ok), "r"(id), "r"(n)
      : "memory");
  return all != 0;
}

// Adds the weights of a unit's 128 columns to a key's four partial sums; MASKED: only those of columns
// c_min .. c_min + c_n - 1.  The next 32 columns are on their way from tensor memory while 32 are
// worked on (in straight-line code: what a load writes must not be touched before its wait, not even
// by a copy at the end of a loop's body).
template <bool MASKED>
__device__ __forceinline__ void add_unit(uint32_t tmem, const float* lse, float scale_log2, int c_min, uint32_t c_n,
                                         uint64_t* empty, float2 (&acc)[4]) {
  const float2 scale2 = make_float2(scale_log2, scale_log2);
  uint32_t su[2][32];
  tmem_ld32(tmem, su[0]);
#pragma unroll
  for (int c = 0; c < ST_COLS; c += 32) {
    tmem_ld_wait();
    if (c + 32 < ST_COLS) {
      tmem_ld32(tmem + c + 32, su[(c / 32 + 1) & 1]);
    } else {
      fence_before_sync();
      mbar_arrive(empty);
    }
    const uint32_t* s = su[(c / 32) & 1];
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 l = *(const float4*)&lse[c + j];
      float2 x[2] = {__ffma2_rn(make_float2(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), scale2, make_float2(l.x, l.y)),
                     __ffma2_rn(make_float2(__uint_as_float(s[j + 2]), __uint_as_float(s[j + 3])), scale2, make_float2(l.z, l.w))};
      if (MASKED) {
        const uint32_t at = (uint32_t)(c + j - c_min);
        x[0].x = at < c_n ? x[0].x : -INFINITY;
        x[0].y = at + 1 < c_n ? x[0].y : -INFINITY;
        x[1].x = at + 2 < c_n ? x[1].x : -INFINITY;
        x[1].y = at + 3 < c_n ? x[1].y : -INFINITY;
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        float2& a = acc[((j >> 1) + p) & 3];
        a = __fadd2_rn(a, make_float2(ex2(x[p].x), ex2(x[p].y)));
      }
    }
  }
}

struct SumsWork {
  const int* cu_seqlens;
  const int* ctx_lens;
  int B, nkv, n_rep, key_tiles, tile_tokens;      // key_tiles: of the longest context
  int places;                                     // that a row of the page table has: no sequence is longer
  __device__ __forceinline__ int length(int b) const { return min(ctx_lens[b], places); }
};
// Query tiles that see a key of tile kt of sequence b.
__device__ __forceinline__ int query_tiles(const SumsWork& w, int b, int kt) {
  const int L = w.length(b), n_new = w.cu_seqlens[b + 1] - w.cu_seqlens[b];
  if (kt * ST_KEYS >= L || n_new <= 0) return 0;
  return (n_new - max(0, kt * ST_KEYS - (L - n_new)) + w.tile_tokens - 1) / w.tile_tokens;
}

// The walk over a CTA's share of the list, which every role makes for itself.
struct Segment {
  int b, kt, g, t0, n;       // sequence, key tile, KV head, first query tile, number of them
  int all;                   // query tiles of these keys
  int unit;                  // number of the segment's first unit
  int left;                  // units of the share from the segment's first on
  int tok0, n_new, start, L; // the sequence: first token of the step, tokens, their first place, length
  __device__ __forceinline__ void load(const SumsWork& w) {
    tok0 = w.cu_seqlens[b];
    n_new = w.cu_seqlens[b + 1] - tok0;
    L = w.length(b);
    start = L - n_new;
  }
  __device__ __forceinline__ bool next(const SumsWork& w) {
    unit += n;
    left -= n;
    if (left <= 0) return false;
    t0 = 0;                                      // (a segment takes all that is left of its keys' query tiles)
    if (++g == w.nkv) {
      g = 0;
      do {
        if (++kt == w.key_tiles) { kt = 0; ++b; }
        if (b >= w.B) return false;
        all = query_tiles(w, b, kt);
      } while (all == 0);
      load(w);
    }
    n = min(all, left);
    return true;
  }
  __device__ __forceinline__ int key0() const { return kt * ST_KEYS; }
  __device__ __forceinline__ int token(const SumsWork& w, int i) const {     // the first token of query tile t0 + i
    return max(0, key0() - start) + (t0 + i) * w.tile_tokens;
  }
  // the first of the segment's query tiles in which a query sees a key of half `half` (n: none does)
  __device__ __forceinline__ int first_of(const SumsWork& w, int half) const {
    if (half == 0) return 0;
    const int k0 = key0() + 128, need = k0 + 1 - start - max(0, key0() - start);     // tokens of the tiles up to it
    if (k0 >= L) return n;
    return min(n, max(0, (need + w.tile_tokens - 1) / w.tile_tokens - 1 - t0));
  }
};

template <int HD>
__global__ void __launch_bounds__(ST_THREADS, 1)
prefill_sums_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_q, const SumsWork work,
                    const float* lse, float scale_log2, const SumsTarget t, float* part, int* tickets,
                    unsigned long long wait_ns, int starve, int late_trigger) {
  using W = StCfg<HD>;
  constexpr int NS = W::STAGES;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ __align__(16) float s_lse[8][2][ST_COLS];       // [warp][buffer] minus the columns' log-sums, -inf for no row
  __shared__ __align__(8) uint64_t bars[4 + 2 * NS + 8];
  __shared__ int s_scan[ST_THREADS / 32], s_found[4];
  __shared__ uint32_t tmem_holder;
  __shared__ int failed, s_last;
  uint64_t *k_full = bars, *k_empty = bars + 2, *q_full = bars + 4, *q_empty = q_full + NS, *s_full = q_empty + NS,
           *s_empty = s_full + 4;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // ---- the share: units [u0, u1) of U, and where u0 lies (from the step's lengths, which the host
  // wrote before the step's first kernel: all this runs ahead of the dependency wait) ----
  const int pairs = work.B * work.key_tiles, chunk = (pairs + ST_THREADS - 1) / ST_THREADS;
  const int p0 = min(tid * chunk, pairs), p1 = min(p0 + chunk, pairs);
  int mine = 0;
  for (int p = p0; p < p1; ++p) mine += query_tiles(work, p / work.key_tiles, p % work.key_tiles) * work.nkv;
  int before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  if (lane == 31) s_scan[warp] = before;
  if (tid == 0) {
    s_found[0] = -1;
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full + i, 1);
      mbar_init(k_empty + i, 1);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(s_empty + i, 128);
    }
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  int U = 0;
  before -= mine;
  for (int i = 0; i < ST_THREADS / 32; ++i) {
    before += i < warp ? s_scan[i] : 0;
    U += s_scan[i];
  }
  const int per = (U + (int)gridDim.x - 1) / (int)gridDim.x;
  const int u0 = blockIdx.x * per, u1 = min(U, u0 + per);
  if (u0 >= u1) {                                            // (the whole CTA; nothing is allocated yet)
    pdl_wait();
    return;
  }
  if (u0 >= before && u0 < before + mine) {
    int at = before, p = p0, n = 0;
    for (;; ++p) {
      n = query_tiles(work, p / work.key_tiles, p % work.key_tiles);
      if (u0 < at + n * work.nkv) break;
      at += n * work.nkv;
    }
    s_found[0] = p;
    s_found[1] = (u0 - at) / n;                              // KV head
    s_found[2] = (u0 - at) % n;                              // query tile
    s_found[3] = n;
  }
  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t k_s = smem_u32(base), q_s = k_s + 2 * W::K_BYTES;
  const int rows = work.n_rep * work.tile_tokens;
  // columns behind the last row of a query tile are never copied: zeros, so that their scores are finite
  for (int e = tid; e < NS * W::NB * (ST_COLS - rows) * 8; e += ST_THREADS) {
    const int half = e / ((ST_COLS - rows) * 8), in = e - half * ((ST_COLS - rows) * 8);
    *(uint4*)(base + 2 * W::K_BYTES + half * W::Q_HALF + rows * 128 + in * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_async_smem();
  __syncthreads();                                           // s_found is there, and the barriers and zeros are
  Segment sg;
  sg.b = s_found[0] / work.key_tiles;
  sg.kt = s_found[0] % work.key_tiles;
  sg.g = s_found[1];
  sg.t0 = s_found[2];
  sg.all = s_found[3];
  sg.unit = u0;
  sg.left = u1 - u0;
  sg.n = min(sg.all - sg.t0, sg.left);
  sg.load(work);

  const bool copies = warp == ST_COPY_WARP && lane == 0 && !(starve == STARVE_ODD ? blockIdx.x & 1 : starve);
  // the copies of a segment's keys, and of its j-th query tile (number i since the kernel's start)
  auto copy_keys = [&](int s) {
    const int* table = t.page_table + (size_t)sg.b * t.table_width;
    int page[ST_KEYS / WPC_PAGE];                            // (all look-ups on their way before the first is needed)
#pragma unroll
    for (int p = 0; p < ST_KEYS / WPC_PAGE; ++p) {
      const int block = sg.kt * (ST_KEYS / WPC_PAGE) + p;
      page[p] = block * WPC_PAGE < sg.L && block < t.table_width ? table[block] : 0;
    }
    pdl_wait();                                              // (at once after the first time)
    mbar_expect_tx(k_full + (s & 1), W::K_BYTES);
#pragma unroll
    for (int p = 0; p < ST_KEYS / WPC_PAGE; ++p) {
      const int row = (min(max(page[p], 0), t.n_pages - 1) * work.nkv + sg.g) * WPC_PAGE;
#pragma unroll
      for (int hb = 0; hb < W::NB; ++hb)
        tma_load_2d(k_s + (s & 1) * W::K_BYTES + hb * W::K_HALF + p * (WPC_PAGE * 128), &map_k, hb * 64, row, k_full + (s & 1));
    }
  };
  auto copy_queries = [&](int i, int j) {
    const int st = i % NS;
    mbar_expect_tx(q_full + st, rows * 128 * W::NB);
#pragma unroll
    for (int hb = 0; hb < W::NB; ++hb)
      tma_load_3d(q_s + st * W::Q_BYTES + hb * W::Q_HALF, &map_q, hb * 64, sg.g * work.n_rep, sg.tok0 + sg.token(work, j), q_full + st);
  };
  // the first copies start with the dependency wait's end, beside the allocation of tensor memory
  const int primed = min(NS, sg.n);
  if (copies) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
    copy_keys(0);
    for (int j = 0; j < primed; ++j) copy_queries(j, j);
  }
  __syncwarp();
  pdl_wait();
  // (tensor memory only now: the kernel ahead may still need it)
  if (warp == ST_MMA_WARP) tmem_alloc(&tmem_holder, 512);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_holder;
  // (only now: the kernel behind may hold tensor memory while it waits for this one, so every CTA
  // of this one must have got its own first)
  if (!late_trigger) pdl_trigger();
  if (warp == ST_COPY_WARP) {
    if (copies) {
      int s = 0, i = primed;                                 // segments and query tiles so far
      bool ok = true;
      for (;;) {
        for (int j = s == 0 ? primed : 0; j < sg.n; ++j, ++i) {
          ok = mbar_wait(q_empty + i % NS, ((i / NS) & 1) ^ 1, wait_ns);
          if (!ok) break;
          copy_queries(i, j);
        }
        ++s;
        if (!ok || !sg.next(work)) break;
        ok = mbar_wait(k_empty + (s & 1), ((s >> 1) & 1) ^ 1, wait_ns);
        if (!ok) break;
        copy_keys(s);
      }
      if (!ok) atomicExch(&failed, 1);
    }
    if (late_trigger) pdl_trigger();
  } else if (warp == ST_MMA_WARP) {
    if (lane == 0) {
      constexpr uint32_t idesc = instr_desc(ST_COLS, false);
      int s = 0, i = 0, filled[2] = {0, 0};                  // segments, query tiles, scores of each half so far
      bool ok = true;
      do {
        const int first[2] = {0, sg.first_of(work, 1)};
        ok = mbar_wait(k_full + (s & 1), (s >> 1) & 1, wait_ns);
        for (int j = 0; ok && j < sg.n; ++j, ++i) {
          const int st = i % NS;
          ok = mbar_wait(q_full + st, (i / NS) & 1, wait_ns);
          if (!ok) break;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (j < first[half]) continue;
            const int bb = filled[half] & 1;
            ok = ok && mbar_wait(s_empty + half * 2 + bb, ((filled[half] >> 1) & 1) ^ 1, wait_ns);
            if (!ok) break;
            ++filled[half];
            fence_after_sync();
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
              const uint32_t ka = k_s + (s & 1) * W::K_BYTES + (kk >> 2) * W::K_HALF + half * (128 * 128) + (kk & 3) * 32;
              const uint32_t qa = q_s + st * W::Q_BYTES + (kk >> 2) * W::Q_HALF + (kk & 3) * 32;
              umma_bf16(tmem + half * 256 + bb * ST_COLS, smem_desc(ka, 16), smem_desc(qa, 16), idesc, kk > 0 ? 1u : 0u);
            }
            umma_commit(s_full + half * 2 + bb);
          }
          umma_commit(q_empty + st);
        }
        if (ok) umma_commit(k_empty + (s & 1));
        ++s;
      } while (ok && sg.next(work));
      if (!ok) atomicExch(&failed, 1);
    }
  } else {
    // ---- thread r of half `half` owns key key0 + 128 half + r; every warp goes its own pace ----
    const int half = warp >> 2, r = tid & 127;
    const uint32_t at = tmem + half * 256 + ((uint32_t)((warp & 3) * 32) << 16);
    const int nh = work.nkv * work.n_rep;
    // the lane's four columns: their places in a tile's rows of lse, and their tokens
    int col_at[4], col_tok[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = lane * 4 + j;
      col_tok[j] = col < rows ? col / work.n_rep : 1 << 30;
      col_at[j] = (col / work.n_rep) * nh + col % work.n_rep;
    }
    int filled = 0;                                          // units of this half so far
    bool ok = true, more = true;
    while (more) {
      if (tid == 0 && sg.kt == 0 && sg.t0 == 0 && sg.g == 0) check_length(t, work.ctx_lens[sg.b], work.key_tiles * ST_KEYS);
      const int key = sg.key0() + half * 128 + r;
      const int i0 = sg.first_of(work, half);
      int tile_first = sg.token(work, i0);                   // first token of the next query tile
      const float* from = lse + (size_t)(sg.tok0 + tile_first) * nh + sg.g * work.n_rep;
      auto lse_next = [&]() {                                // of that tile's columns, -inf for no row
        const int left = sg.n_new - tile_first;
        float4 v;
        v.x = col_tok[0] < left ? -from[col_at[0]] : -INFINITY;
        v.y = col_tok[1] < left ? -from[col_at[1]] : -INFINITY;
        v.z = col_tok[2] < left ? -from[col_at[2]] : -INFINITY;
        v.w = col_tok[3] < left ? -from[col_at[3]] : -INFINITY;
        return v;
      };
      float2 acc[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      float4 next_lse = lse_next();
      for (int i = i0; ok && i < sg.n; ++i) {
        const float4 my_lse = next_lse;
        const int first_tok = tile_first;
        tile_first += work.tile_tokens;
        from += work.tile_tokens * nh;
        next_lse = lse_next();
        const int bb = filled & 1;
        *(float4*)&s_lse[warp][bb][lane * 4] = my_lse;
        __syncwarp();
        ok = mbar_wait(s_full + half * 2 + bb, (filled >> 1) & 1, wait_ns);
        ok = __all_sync(0xffffffffu, ok);
        ++filled;
        if (!ok) break;
        fence_after_sync();
        const float* cl = s_lse[warp][bb];
        // keys that not every query sees, or columns that are no rows of this sequence: the key is seen
        // by columns c_min .. c_min + c_n - 1
        if (key - r + 127 > sg.start + first_tok || tile_first > sg.n_new) {
          const int c_min = max(key - sg.start - first_tok, 0) * work.n_rep;
          const int c_n = max(min(sg.n_new - first_tok, work.tile_tokens) * work.n_rep - c_min, 0);
          add_unit<true>(at + bb * ST_COLS, cl, scale_log2, c_min, (uint32_t)c_n, s_empty + half * 2 + bb, acc);
        } else {
          add_unit<false>(at + bb * ST_COLS, cl, scale_log2, 0, 0u, s_empty + half * 2 + bb, acc);
        }
      }
      float w = ((acc[0].x + acc[0].y) + (acc[1].x + acc[1].y)) + ((acc[2].x + acc[2].y) + (acc[3].x + acc[3].y));
      // ---- the end of a segment (both halves meet here, whatever became of their waits; after one that ran
      // out the CTA walks the rest of its share without waiting or adding, for the tickets alone) ----
      bool adds;
      if (sg.n == sg.all) {
        adds = ok = all_of(3, 256, ok);
      } else {
        // The keys' units are [first, first + all): this CTA's part goes to its slot 0 if it is the
        // first segment of its share, else to slot 1 (it is the last one then).
        const int first = sg.unit - sg.t0;
        part[(size_t)(2 * blockIdx.x + (sg.unit == u0 ? 0 : 1)) * ST_KEYS + half * 128 + r] = w;
        __threadfence();
        ok = all_of(3, 256, ok);
        const int c0 = first / per, c1 = (first + sg.all - 1) / per;
        if (tid == 0) {
          int* ticket = tickets + (sg.b * work.key_tiles + sg.kt) * work.nkv + sg.g;
          const int taken = atomicAdd(ticket, ok ? 1 : ST_FAILED + 1);
          const bool last = (taken & (ST_FAILED - 1)) == c1 - c0;
          if (last) *ticket = 0;                             // ready for the next launch
          s_last = last && ok && taken < ST_FAILED;          // (with a failed CTA among them nobody adds)
          __threadfence();
        }
        all_of(3, 256, true);
        adds = s_last;
        if (adds) {
          w = 0.f;
          for (int c = c0; c <= c1; c += 8) {                // (eight loads on their way at a time)
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
              v[j] = c + j <= c1 ? __ldcg(part + (size_t)(2 * (c + j) + ((c + j) * per >= first ? 0 : 1)) * ST_KEYS + half * 128 + r) : 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) w += v[j];
          }
        }
        all_of(3, 256, true);                                // (s_last is written again)
      }
      if (adds && key < sg.L)
        add_sum(t, work.nkv, sg.b, sg.g, key, key >= sg.start ? sg.tok0 + key - sg.start : -1, w);
      more = sg.next(work);
    }
    if (!ok) atomicExch(&failed, 1);
  }
  fence_before_sync();
  __syncthreads();
  if (failed) {
    // a wait ran out: give copies and MMAs in flight time to land before shared memory goes away
    if (tid == 0 && t.status) atomicExch(t.status, WPC_ERR_DEVICE_WAIT);
    const unsigned long long now = global_ns();
    while (global_ns() - now < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == ST_MMA_WARP) {
    fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

template <int HD>
static int launch_sums(const void* q, int q_stride, int n_tokens, const void* k_pages, const int* cu_seqlens,
                       const int* ctx_lens, const float* lse, int B, int nh, int nkv, float scale, int max_new,
                       int max_ctx, const SumsTarget& t, float* part, int* tickets, int n_tickets, cudaStream_t stream) {
  static int configured[MAX_DEVICES];
  if (int rc = allow_smem(prefill_sums_kernel<HD>, StCfg<HD>::SMEM, configured)) return rc;
  const int n_rep = nh / nkv, tile_tokens = ST_COLS / n_rep;
  const long cache_rows = (long)t.n_pages * nkv * WPC_PAGE;
  if (cache_rows > 0x7fffffffL) return WPC_ERR_TOO_LARGE;
  const int key_tiles = (max_ctx + ST_KEYS - 1) / ST_KEYS;
  const long keys = (long)B * key_tiles * nkv, units = keys * ((max_new + tile_tokens - 1) / tile_tokens);
  if (units > 0x7fffffffL - 1024) return WPC_ERR_TOO_LARGE;
  if (n_tickets < keys) return WPC_ERR_BAD_ARGUMENT;
  CUtensorMap mk, mq;
  if (int rc = tc::tensor_map(k_pages, (int)cache_rows, HD, HD, WPC_PAGE, &mk)) return rc;
  if (int rc = tc::tensor_map_heads(q, n_tokens, nh, HD, q_stride, tile_tokens, n_rep, &mq)) return rc;
  const SumsWork work{cu_seqlens, ctx_lens, B, nkv, n_rep, key_tiles, tile_tokens, t.table_width * WPC_PAGE};
  const unsigned ctas = (unsigned)(units < sm_count() ? units : sm_count());
  wpc::launch(prefill_sums_kernel<HD>, dim3(ctas), ST_THREADS, StCfg<HD>::SMEM, stream, mk, mq, work, lse,
              scale * 1.4426950408889634f, t, part, tickets, wait_policy().limit_ns, wait_policy().starve,
              max_new >= 1024 ? 1 : 0);
  return launch_status();
}

}  // namespace fatc
}  // namespace wpc

extern "C" {

// Head sizes 64 and 128, at most 128 heads to a group; q rows 16-byte aligned (q_stride a multiple of 8).
// part: float32 [2 * SMs of the device][256]; tickets: B * nkv * ceil(max_ctx / 256) of them, zero
// between launches.
int wpc_weight_sums_tc(const void* q, int q_stride, int n_tokens, const void* k_pages, const int* page_table,
                       int table_width, const int* cu_seqlens, const int* ctx_lens, const int* token_positions,
                       const float* lse, int B, int nh, int nkv, int hd, float scale, int max_new, int max_ctx,
                       int n_pages, float* weight_sums, int* stored_positions, int* status, float* part, int* tickets,
                       int n_tickets, cudaStream_t stream) {
  if (B <= 0 || max_new <= 0 || max_ctx <= 0) return 0;
  if (!wpc_attention_prefill_tc_supports(nh, nkv, hd) || q_stride % 8 || (((uintptr_t)q | (uintptr_t)k_pages) & 15))
    return WPC_ERR_UNSUPPORTED;
  if (!lse || !part || !tickets || n_pages < 1) return WPC_ERR_BAD_ARGUMENT;
  const wpc::SumsTarget t{page_table, table_width, n_pages, token_positions, weight_sums, stored_positions, status};
  if (hd == 128)
    return wpc::fatc::launch_sums<128>(q, q_stride, n_tokens, k_pages, cu_seqlens, ctx_lens, lse, B, nh, nkv, scale,
                                       max_new, max_ctx, t, part, tickets, n_tickets, stream);
  return wpc::fatc::launch_sums<64>(q, q_stride, n_tokens, k_pages, cu_seqlens, ctx_lens, lse, B, nh, nkv, scale,
                                    max_new, max_ctx, t, part, tickets, n_tickets, stream);
}

}  // extern "C"
