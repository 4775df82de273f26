// Causal grouped-query attention of a prompt over the paged cache on the 5th-generation tensor
// cores (wpc-runtime/src/model.rs:476-510 is the arithmetic).
//
// A CTA takes 128 rows of (token, head-in-group) of one sequence and one KV head (or two such
// tiles) and walks the pages (64 keys) that its rows see.  Per page:
//
//   S = Q K^T      tcgen05.mma, Q [128, hd] and the K page [64, hd] in shared memory (K-major,
//                  128-byte swizzle), S [128, 64] float32 in tensor memory
//   softmax        thread r owns row r: tcgen05.ld of its 64 scores, scale, mask, running
//                  maximum and sum in float32, P = exp2(S - m) as bfloat16 back into tensor
//                  memory, over the first 32 columns of the scores that it came from
//   O += P V       tcgen05.mma with the A operand P [128, 64] from tensor memory, the V page
//                  [64, hd] as it lies in the cache (hd contiguous: an MN-major B operand),
//                  O [128, hd] float32 in tensor memory
//
// P is rounded to the values' type, since a matrix instruction takes both operands in one type (at most half a step, 2^-8 of
// a weight, as the rounding of the output); its sums are those of the unrounded weights.
// The running maximum that the exponentials use is only raised when the true maximum has
// grown by more than 8 (a factor 256, harmless in float32); then the thread rescales its row
// of O in tensor memory.  Separate warps copy the pages (TMA), issue the MMAs and do the
// softmax; they meet at mbarriers only (see the kernel).  Every wait is bounded.  head_dim 64
// or 128; other sizes take the mma.sync kernel.
#include <cuda.h>

#include "api.h"
#include "attention_tc.cuh"
#include "common.cuh"
#include "tensor_map.h"

namespace wpc {
namespace fatc {

constexpr int PAGE = WPC_PAGE;
constexpr int THREADS = 128;
constexpr int ROWS = 128;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_STEP = 8.0f;

template <int HD>
struct Cfg {
  static constexpr int NB = HD / 64;                      // 64-wide blocks along head_dim
  static constexpr int Q_BYTES = NB * ROWS * 128;
  static constexpr int PAGE_BYTES = NB * PAGE * 128;      // one K or V page
};

// ---- the kernel -------------------------------------------------------------------------------------
// A CTA takes NT row tiles of 128 rows (NT = 2: 256 rows, one CTA to an SM; NT = 1: two CTAs to
// an SM).  Warps 0 .. 4 NT - 1: one thread per row, softmax only.  The next warp (one thread)
// issues every tcgen05.mma, the last warp (one thread) copies the K and V pages with TMA.
// Nothing in the page loop stops the whole CTA: the roles meet at mbarriers only where data
// passes from one to the other.
//
//   q_full                  softmax threads -> MMA    the Q rows are in shared memory
//   k_full[NS], v_full[NS]  TMA -> MMA                a page has landed (transaction bytes)
//   k_empty[NS], v_empty[NS]  MMA (commit) -> TMA     the MMAs that read the page have finished
//   s_full[NT][2]           MMA (commit) -> softmax   a tile's scores of a page are in tensor memory
//   s_empty[NT][2]          softmax -> MMA            they have been read (128 arrivals)
//   p_full[NT]              softmax -> MMA            P is in tensor memory and O is rescaled (128)
//   p_empty[NT]             MMA (commit) -> softmax   P V of the page has finished: P may be
//                                                     overwritten and O touched
// While the threads do the softmax of page j the tensor pipe computes the scores of page j + 1
// (second score buffer) and the weighted values of page j - 1.  With two row tiles every page
// is copied once for 256 rows (the copies from L2 bound the one-tile kernel at long prompts:
// 32 KiB for 4.2 MFLOP), and the MMAs of the two tiles, which do not depend on one another,
// take turns, so that one tile's chain of accumulations does not leave the pipe idle.  Both
// tiles walk the same pages; a page that one of them does not see is masked for it.
template <int HD, int NT>
struct WsCfg {
  using C = Cfg<HD>;
  static constexpr int NS = NT == 2 ? 4 : 2;              // stages of K and of V
  static constexpr int THREADS = 128 * NT + 64;
  static constexpr int TMEM_COLS = NT == 2 ? 512 : 256;   // per tile: two score buffers of 64 and HD for O
  static constexpr int N_BARS = 1 + 4 * NS + 6 * NT;
  // 896 bytes of slack bring the 128-byte aligned start to a 1024-byte boundary; with one tile
  // two CTAs fit an SM (tensor memory allows no third: 2 x 256 columns)
  static constexpr int SMEM = 896 + NT * C::Q_BYTES + 2 * NS * C::PAGE_BYTES + N_BARS * 8 + 8;
};

// Three forms, compiled on their own (the ordinary one carries nothing of the others; with their code
// behind run-time tests prefill of 8,192 tokens lost 2 %):
//   PF_PLAIN  all earlier positions, or a window of them
//   PF_SINKS  beside its window a query sees the first `sinks` positions.  Their pages that lie before
//             the window's first page come first; pages are counted in one range (attention_mma.cuh)
//   PF_SUMS   lse gets each row's maximum + log2(sum) in units of log 2, for the sums of weights
//             (attention_sums_tc.cu)
// PF_SHARED beside one of the last two: several CTAs (n_splits) share a row tile's pages, for a chunk of few
// tokens over a long cache, whose tiles leave SMs idle.  Each leaves its unnormalised output, maximum and
// sum in its slot of part_o and part_ml, and prefill_join_kernel adds them in order.
// (A form of its own too: as a run-time choice in the others it cost prompts of 2,048 tokens 1 to 3 %.  64 tokens
// of the 7B shape over 16,384 positions with their sums: 248 -> 60 us.)
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
constexpr int PF_PLAIN = 0, PF_SINKS = 1, PF_SUMS = 2, PF_SHARED = 4;

template <int HD, int NT, int MODE>
__global__ void __launch_bounds__(WsCfg<HD, NT>::THREADS, NT == 2 ? 1 : 2)
prefill_ws_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const __nv_bfloat16* __restrict__ q, int q_stride, __nv_bfloat16* __restrict__ out, int out_stride,
                  const int* __restrict__ page_table, int table_width, const int* __restrict__ cu_seqlens,
                  const int* __restrict__ ctx_lens, int nh, int nkv, float scale_log2, int window,
                  int* __restrict__ status, unsigned long long wait_ns, int starve, int n_sm, int late_trigger,
                  int sinks, float* __restrict__ lse, int n_splits, float4* __restrict__ part_o,
                  float2* __restrict__ part_ml) {
  using C = Cfg<HD>;
  using W = WsCfg<HD, NT>;
  constexpr bool SINKS = (MODE & PF_SINKS) != 0, SHARED = (MODE & PF_SHARED) != 0;
  static_assert(!SHARED || NT == 1, "a shared tile is one row tile");
  constexpr int NS = W::NS;
  constexpr int TROWS = NT * ROWS;
  if (!late_trigger) pdl_trigger();
  pdl_wait();
  extern __shared__ __align__(128) uint8_t smem_raw[];
  // The last tiles of a sequence see the most keys: they start first, and for all KV heads
  // before any lighter tile (the KV head is the fastest grid index), so that no heavy tile is
  // left for the end.  An SM takes new CTAs of this kernel in turn: while the older of its two
  // CTAs runs, the place of the younger one, once it has ended, stays empty (seen in a trace of
  // start and end times; without tcgen05.relinquish_alloc_permit an SM even runs one CTA at a
  // time).  So the two CTAs that an SM gets at the start should be equally heavy: the device
  // hands the first n_sm CTAs of a grid to one SM each and the next n_sm to the same SMs in
  // the same order, and position p of the grid takes rank 2 p, or 2 (p - n_sm) + 1, of the
  // pieces in descending order (one sequence only; 53.7 -> 47.3 us at 2,048 tokens of the 7B shape).
  int rank = (int)(blockIdx.y * gridDim.x + blockIdx.x);
  if (gridDim.z == 1) {
    const int n = (int)(gridDim.x * gridDim.y), two = n - n_sm < n_sm ? n - n_sm : n_sm;   // SMs that get two at the start
    if (two > 0) {
      if (rank < n_sm) rank = rank < two ? 2 * rank : rank + two;
      else if (rank < 2 * n_sm) rank = 2 * (rank - n_sm) + 1;
    }
  }
  const int tile = (int)gridDim.y - 1 - rank / (int)gridDim.x, g = rank % (int)gridDim.x;
  const int b = SHARED ? blockIdx.z / n_splits : blockIdx.z, split = SHARED ? blockIdx.z % n_splits : 0;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n_rep = nh / nkv;
  const int tok0 = cu_seqlens[b];
  const int n_new = cu_seqlens[b + 1] - tok0;
  const int n_rows = n_new * n_rep;
  const int row0 = tile * TROWS;
  if (row0 >= n_rows) return;                         // whole CTA, before anything is allocated

  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t q_s = smem_u32(base);                                 // [NT] tiles of Q
  const uint32_t k_s = q_s + NT * C::Q_BYTES;                          // [NS] pages
  const uint32_t v_s = k_s + NS * C::PAGE_BYTES;                       // [NS] pages
  uint64_t* bars = (uint64_t*)(base + NT * C::Q_BYTES + 2 * NS * C::PAGE_BYTES);
  uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = k_full + NS, *v_full = k_empty + NS, *v_empty = v_full + NS,
           *s_full = v_empty + NS /* [NT][2] */, *s_empty = s_full + 2 * NT, *p_full = s_empty + 2 * NT,
           *p_empty = p_full + NT;
  uint32_t* tmem_holder = (uint32_t*)(p_empty + NT);
  int* failed = (int*)(tmem_holder + 1);
  constexpr int MMA_WARP = 4 * NT, COPY_WARP = 4 * NT + 1;

  if (tid == 0) {
    mbar_init(q_full, 128 * NT);
    for (int i = 0; i < NS; ++i) {
      mbar_init(k_full + i, 1);
      mbar_init(k_empty + i, 1);
      mbar_init(v_full + i, 1);
      mbar_init(v_empty + i, 1);
    }
    for (int i = 0; i < 2 * NT; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(s_empty + i, 128);
    }
    for (int i = 0; i < NT; ++i) {
      mbar_init(p_full + i, 128);
      mbar_init(p_empty + i, 1);
    }
    *failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) tmem_alloc(tmem_holder, W::TMEM_COLS);

  // (PF_PLAIN takes the caller's word that the page table has a place for every position)
  const int L = MODE == PF_PLAIN ? ctx_lens[b] : min(ctx_lens[b], table_width * PAGE);
  const int start = L - n_new;
  const int* table = page_table + (size_t)b * table_width;
  // pages that any row of the CTA sees: from the window start of its first row to the position of its last
  const int last_row = min(row0 + TROWS - 1, n_rows - 1);
  const int tile_pos_hi = start + last_row / n_rep;
  const int tile_pos_lo = start + row0 / n_rep;
  const int tile_lo = (window > 0 && tile_pos_lo - window + 1 > 0) ? tile_pos_lo - window + 1 : 0;
  const int first = tile_lo / PAGE, ns = SINKS ? min((sinks + PAGE - 1) / PAGE, first) : 0;
  const int blk0 = first - ns, blk1 = tile_pos_hi / PAGE + 1;
  const int all_pg = blk1 - blk0;
  // this CTA's share of the tile's list of pages (a tile of few pages leaves some shares empty)
  const int j0 = SHARED ? (int)((long)all_pg * split / n_splits) : 0;
  const int n_pg = SHARED ? (int)((long)all_pg * (split + 1) / n_splits) - j0 : all_pg;
  auto block = [&](int j) { return SINKS && j0 + j < ns ? j0 + j : blk0 + j0 + j; };   // page j of the CTA's share

  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem_base = *tmem_holder;
  // tile t: scores in columns t * 128 .. + 127 (two buffers of 64), O in columns NT * 128 + t * HD ..
  auto tmem_S = [&](int t, int bb) { return tmem_base + t * 128 + bb * 64; };
  auto tmem_O = [&](int t) { return tmem_base + NT * 128 + t * HD; };

  if (warp == COPY_WARP) {
    // ---- copies (none with `starve`, the tests' way to make the waits below run out) ----
    if (lane == 0 && !starve) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
      int page_next = SHARED && n_pg <= 0 ? 0 : max(table[block(0)], 0);
      for (int j = 0; j < n_pg; ++j) {
        const int st = j % NS, n = j / NS;
        const int row = (page_next * nkv + g) * PAGE;
        if (j + 1 < n_pg) page_next = max(table[block(j + 1)], 0);
        if (!mbar_wait(k_empty + st, (n & 1) ^ 1, wait_ns)) { atomicExch(failed, 1); break; }
        mbar_expect_tx(k_full + st, C::PAGE_BYTES);
#pragma unroll
        for (int hb = 0; hb < C::NB; ++hb)
          tma_load_2d(k_s + st * C::PAGE_BYTES + hb * (PAGE * 128), &map_k, hb * 64, row, k_full + st);
        if (!mbar_wait(v_empty + st, (n & 1) ^ 1, wait_ns)) { atomicExch(failed, 1); break; }
        mbar_expect_tx(v_full + st, C::PAGE_BYTES);
#pragma unroll
        for (int hb = 0; hb < C::NB; ++hb)
          tma_load_2d(v_s + st * C::PAGE_BYTES + hb * (PAGE * 128), &map_v, hb * 64, row, v_full + st);
      }
    }
    // a long prompt's kernel lets the kernel after it go only now, when this CTA's copies are all
    // on their way (its CTAs would otherwise sit on SMs that this kernel still needs)
    if (late_trigger) pdl_trigger();
  } else if (warp == MMA_WARP) {
    // ---- MMA issue ----
    if (lane == 0) {
      constexpr uint32_t idesc_qk = instr_desc(64, false);
      constexpr uint32_t idesc_pv = instr_desc(HD, true);
      // the scores of page j for all tiles, the tiles taking turns
      auto issue_qk = [&](int j) {
        fence_after_sync();
        const uint32_t kb = k_s + (j % NS) * C::PAGE_BYTES;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t ka = kb + (kk >> 2) * (PAGE * 128) + (kk & 3) * 32;
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const uint32_t qa = q_s + t * C::Q_BYTES + (kk >> 2) * (ROWS * 128) + (kk & 3) * 32;
            umma_bf16(tmem_S(t, j & 1), smem_desc(qa, 16), smem_desc(ka, 16), idesc_qk, kk > 0 ? 1u : 0u);
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) umma_commit(s_full + t * 2 + (j & 1));
        umma_commit(k_empty + j % NS);
      };
      bool ok = (SHARED && n_pg <= 0) || (mbar_wait(q_full, 0, wait_ns) && mbar_wait(k_full, 0, wait_ns));
      if (ok && !(SHARED && n_pg <= 0)) issue_qk(0);
      for (int j = 0; ok && j < n_pg; ++j) {
        if (j + 1 < n_pg) {
          const int j1 = j + 1;
          ok = mbar_wait(k_full + j1 % NS, (j1 / NS) & 1, wait_ns);
#pragma unroll
          for (int t = 0; t < NT; ++t) ok = ok && mbar_wait(s_empty + t * 2 + (j1 & 1), ((j1 >> 1) & 1) ^ 1, wait_ns);
          if (!ok) break;
          issue_qk(j1);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) ok = ok && mbar_wait(p_full + t, j & 1, wait_ns);
        ok = ok && mbar_wait(v_full + j % NS, (j / NS) & 1, wait_ns);
        if (!ok) break;
        fence_after_sync();
        const uint32_t vb = v_s + (j % NS) * C::PAGE_BYTES;
#pragma unroll
        for (int kc = 0; kc < PAGE / 16; ++kc) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
            umma_bf16_ts(tmem_O(t), tmem_S(t, j & 1) + kc * 8, smem_desc(vb + kc * 2048, PAGE * 128),
                      idesc_pv, (j > 0 || kc > 0) ? 1u : 0u);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) umma_commit(p_empty + t);
        umma_commit(v_empty + j % NS);
      }
      if (!ok) atomicExch(failed, 1);
    }
  } else {
    // ---- softmax: thread (t, rt) owns row row0 + t * 128 + rt of tile t ----
    const int t = warp >> 2, rt = tid & 127;
    const int r = row0 + t * ROWS + rt;
    const bool valid = r < n_rows;
    const int t_row = valid ? r / n_rep : 0;
    const int h_row = g * n_rep + (valid ? r % n_rep : 0);
    const int p_row = start + t_row;
    const int lo_row = (window > 0 && p_row - window + 1 > 0) ? p_row - window + 1 : 0;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    {
      const __nv_bfloat16* src = after_wait(q) + (size_t)(tok0 + t_row) * q_stride + (size_t)h_row * HD;
      uint8_t* my_q = base + t * C::Q_BYTES;
      // (all loads ahead of the first store, which they cannot be moved across: with loads and stores by turns
      // 2,048 tokens of the 7B shape took 41.4 us, not 39.6)
      uint4 v[HD / 8];
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) v[c] = valid ? *(const uint4*)(src + c * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) *(uint4*)(my_q + (c >> 3) * (ROWS * 128) + swz(rt, c & 7)) = v[c];
      fence_async_smem();
      mbar_arrive(q_full);
    }
    float m_used = -INFINITY, l_sum = 0.f;
    bool ok = true;
    for (int j = 0; j < n_pg; ++j) {
      const int bb = j & 1;
      ok = mbar_wait(s_full + t * 2 + bb, (j >> 1) & 1, wait_ns);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      fence_after_sync();
      uint32_t su[64];
      tmem_ld32(tmem_S(t, bb) + lane_off, su);
      tmem_ld32(tmem_S(t, bb) + lane_off + 32, su + 32);
      tmem_ld_wait();
      fence_before_sync();
      mbar_arrive(s_empty + t * 2 + bb);                   // the score buffer may be overwritten
      const int abs0 = block(j) * PAGE;
      // four partial maxima (and sums below): a single running value would be a chain of 64
      // dependent instructions.  Only pages that this row does not see whole are masked.
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (valid && abs0 + PAGE - 1 <= p_row && (abs0 >= lo_row || (SINKS && abs0 + PAGE <= sinks))) {
#pragma unroll
        for (int i = 0; i < 64; i += 8) {                  // (pairs of values to a maximum: one three-input instruction)
          mx4[0] = fmaxf(fmaxf(mx4[0], __uint_as_float(su[i])), __uint_as_float(su[i + 1]));
          mx4[1] = fmaxf(fmaxf(mx4[1], __uint_as_float(su[i + 2])), __uint_as_float(su[i + 3]));
          mx4[2] = fmaxf(fmaxf(mx4[2], __uint_as_float(su[i + 4])), __uint_as_float(su[i + 5]));
          mx4[3] = fmaxf(fmaxf(mx4[3], __uint_as_float(su[i + 6])), __uint_as_float(su[i + 7]));
        }
      } else if (MODE != PF_PLAIN) {
        // (the keys that are seen as bits: with three comparisons a score PF_SINKS needed every register
        // and spilled; 157 against 143 us at 2,048 tokens of 8 Ki, window 4,096)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k0 = abs0 + h * 32;
          const uint32_t seen = valid ? low_bits(p_row - k0 + 1) & (~low_bits(lo_row - k0) | (SINKS ? low_bits(sinks - k0) : 0u)) : 0u;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float sc = seen >> i & 1 ? __uint_as_float(su[h * 32 + i]) : -INFINITY;
            su[h * 32 + i] = __float_as_uint(sc);
            mx4[i & 3] = fmaxf(mx4[i & 3], sc);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          const int kabs = abs0 + i;
          const float sc = (valid && kabs >= lo_row && kabs <= p_row) ? __uint_as_float(su[i]) : -INFINITY;
          su[i] = __float_as_uint(sc);
          mx4[i & 3] = fmaxf(mx4[i & 3], sc);
        }
      }
      float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      mx *= scale_log2;
      // raise the maximum in use only when the true one has outgrown it
      float alpha = 1.f;
      bool rescale = false;
      if (mx > m_used + RESCALE_STEP || (m_used == -INFINITY && mx > -INFINITY)) {
        alpha = (m_used == -INFINITY) ? 0.f : exp2f(m_used - mx);
        rescale = m_used != -INFINITY;
        m_used = mx;
      }
      l_sum *= alpha;
      const float neg_m = (m_used == -INFINITY) ? 0.f : -m_used;     // all scores are -inf then: p = 0
      // (two values to an instruction where there is one: fma.f32x2, add.f32x2)
      const float2 scale2 = make_float2(scale_log2, scale_log2), neg_m2 = make_float2(neg_m, neg_m);
      float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      uint32_t pw[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float2 x = __ffma2_rn(make_float2(__uint_as_float(su[2 * i]), __uint_as_float(su[2 * i + 1])), scale2, neg_m2);
        const float2 pr = make_float2(ex2(x.x), ex2(x.y));
        sum2[i & 1] = __fadd2_rn(sum2[i & 1], pr);
        const __nv_bfloat162 pb = __floats2bfloat162_rn(pr.x, pr.y);
        pw[i] = *(const uint32_t*)&pb;
      }
      l_sum += (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
      // the weighted values of the page before must be done before O and P are touched
      if (j > 0) {
        ok = mbar_wait(p_empty + t, (j - 1) & 1, wait_ns);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_after_sync();
      }
      if (__any_sync(0xffffffffu, rescale)) {
        // the whole warp takes part (tcgen05.ld/st are warp-wide); rows that keep their maximum use 1
        const float a = rescale ? alpha : 1.f;
#pragma unroll
        for (int c = 0; c < HD; c += 32) {
          uint32_t ou[32];
          tmem_ld32(tmem_O(t) + lane_off + c, ou);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) ou[i] = __float_as_uint(__uint_as_float(ou[i]) * a);
          tmem_st32(tmem_O(t) + lane_off + c, ou);
        }
        tmem_st_wait();
      }
      // P goes back into tensor memory, over the first 32 columns of the scores that it came
      // from (two bfloat16 a column): P V takes its A operand from there.  The MMAs that wrote
      // those columns and the one that read the weights of two pages ago are done (the scores'
      // barrier came after them); the scores of the page after next, which will overwrite them,
      // are issued after this page's P V and run after it.
      tmem_st32(tmem_S(t, bb) + lane_off, pw);
      tmem_st_wait();
      if (MODE != PF_PLAIN && abs0 + PAGE > L) {
        // behind the end of the sequence lies what the page's last owner left: a weight of zero
        // times an infinity would be no zero, so those value rows are cleared before P V
        ok = mbar_wait(v_full + j % NS, (j / NS) & 1, wait_ns);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        uint8_t* v_page = base + NT * C::Q_BYTES + (NS + j % NS) * C::PAGE_BYTES;
        for (int e = rt + (L - abs0) * 8; e < PAGE * 8; e += ROWS)
#pragma unroll
          for (int hb = 0; hb < C::NB; ++hb) *(uint4*)(v_page + hb * (PAGE * 128) + e * 16) = make_uint4(0, 0, 0, 0);
        fence_async_smem();
      }
      fence_before_sync();
      mbar_arrive(p_full + t);
    }
    if (ok && !(SHARED && n_pg <= 0)) {
      ok = mbar_wait(p_empty + t, (n_pg - 1) & 1, wait_ns);
      ok = __all_sync(0xffffffffu, ok);
      fence_after_sync();
    }
    if (!ok) atomicExch(failed, 1);
    if constexpr (SHARED) {
      // slot [HD / 4][128 rows] of four values: neighbouring rows lie side by side
      const size_t slot = ((size_t)blockIdx.z * gridDim.y + tile) * gridDim.x + g;
      if (valid) part_ml[slot * ROWS + rt] = make_float2(m_used, ok ? l_sum : -1.f);      // (-1: a wait ran out)
      if (ok && n_pg > 0) {
#pragma unroll
        for (int c = 0; c < HD; c += 32) {
          uint32_t ou[32];
          tmem_ld32(tmem_O(t) + lane_off + c, ou);
          tmem_ld_wait();
          if (valid)
#pragma unroll
            for (int jj = 0; jj < 32; jj += 4)
              part_o[(slot * (HD / 4) + (c + jj) / 4) * ROWS + rt] =
                  make_float4(__uint_as_float(ou[jj]), __uint_as_float(ou[jj + 1]), __uint_as_float(ou[jj + 2]), __uint_as_float(ou[jj + 3]));
        }
      }
    } else if (ok) {
      const float inv = l_sum > 0.f ? 1.f / l_sum : 0.f;
      if ((MODE & PF_SUMS) && valid) lse[(size_t)(tok0 + t_row) * nh + h_row] = m_used + log2f(l_sum);
      __nv_bfloat16* dst = out + (size_t)(tok0 + t_row) * out_stride + (size_t)h_row * HD;
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        uint32_t ou[32];
        tmem_ld32(tmem_O(t) + lane_off + c, ou);
        tmem_ld_wait();
        if (valid) {
#pragma unroll
          for (int jj = 0; jj < 32; jj += 8) {
            uint4 o;
            __nv_bfloat162 a0 = __floats2bfloat162_rn(__uint_as_float(ou[jj]) * inv, __uint_as_float(ou[jj + 1]) * inv);
            __nv_bfloat162 a1 = __floats2bfloat162_rn(__uint_as_float(ou[jj + 2]) * inv, __uint_as_float(ou[jj + 3]) * inv);
            __nv_bfloat162 a2 = __floats2bfloat162_rn(__uint_as_float(ou[jj + 4]) * inv, __uint_as_float(ou[jj + 5]) * inv);
            __nv_bfloat162 a3 = __floats2bfloat162_rn(__uint_as_float(ou[jj + 6]) * inv, __uint_as_float(ou[jj + 7]) * inv);
            o.x = *(uint32_t*)&a0; o.y = *(uint32_t*)&a1; o.z = *(uint32_t*)&a2; o.w = *(uint32_t*)&a3;
            *(uint4*)(dst + c + jj) = o;
          }
        }
      }
    } else if ((MODE & PF_SUMS) && valid) {
      // (a wait ran out: the row's weights count as nothing, so the sums of earlier entries take no harm)
      lse[(size_t)(tok0 + t_row) * nh + h_row] = INFINITY;
    }
  }
  fence_before_sync();
  __syncthreads();
  if (*failed) {
    // a wait ran out: give copies in flight time to land before shared memory goes away
    if (tid == 0 && status) atomicExch(status, WPC_ERR_DEVICE_WAIT);
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == MMA_WARP) {
    fence_after_sync();
    tmem_dealloc(tmem_base, W::TMEM_COLS);
  }
}

// Joins the shares of a row tile: a thread to a row and JOIN of its values.  Reads what the shares wrote, from L2,
// 16 bytes a thread with a warp's rows side by side (outputs laid out by rows instead: 512 tokens in two shares
// 29.8 us against 24.6); with one share's loads at a time the join of 16 shares took 5 us longer.  Grid as the
// shared kernel's, with HD / JOIN blocks to a tile in place of its shares.
constexpr int JOIN = 16;
template <int HD>
__global__ void __launch_bounds__(ROWS)
prefill_join_kernel(const float4* part_o, const float2* part_ml, __nv_bfloat16* __restrict__ out, int out_stride,
                    float* __restrict__ lse, const int* cu_seqlens, int nh, int nkv, int n_splits) {
  constexpr int PARTS = HD / JOIN;
  pdl_trigger();
  pdl_wait();
  const int g = blockIdx.x, tile = blockIdx.y, b = blockIdx.z / PARTS, part = blockIdx.z % PARTS, rt = threadIdx.x;
  const int n_rep = nh / nkv, tok0 = cu_seqlens[b], r = tile * ROWS + rt;
  if (r >= (cu_seqlens[b + 1] - tok0) * n_rep) return;
  auto slot = [&](int s) { return ((size_t)(b * n_splits + s) * gridDim.y + tile) * gridDim.x + g; };
  float m = -INFINITY;
#pragma unroll 4
  for (int s = 0; s < n_splits; ++s) m = fmaxf(m, part_ml[slot(s) * ROWS + rt].x);
  float den = 0.f, num[JOIN] = {};
  bool lost = false;
  for (int s0 = 0; s0 < n_splits; s0 += 4) {               // (four shares' loads on their way at once)
    float2 ml[4];
    float4 o[4][JOIN / 4];
#pragma unroll
    for (int k = 0; k < 4; ++k) ml[k] = s0 + k < n_splits ? part_ml[slot(s0 + k) * ROWS + rt] : make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < JOIN / 4; ++i)                   // (a sum of 0: no page, or nothing of it seen; its output may not be written)
        o[k][i] = ml[k].y != 0.f ? part_o[(slot(s0 + k) * (HD / 4) + part * (JOIN / 4) + i) * ROWS + rt] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      lost |= ml[k].y < 0.f;
      const float f = ml[k].y != 0.f ? exp2f(ml[k].x - m) : 0.f;
      den = fmaf(f, ml[k].y, den);
#pragma unroll
      for (int i = 0; i < JOIN / 4; ++i) {
        num[4 * i] = fmaf(f, o[k][i].x, num[4 * i]);
        num[4 * i + 1] = fmaf(f, o[k][i].y, num[4 * i + 1]);
        num[4 * i + 2] = fmaf(f, o[k][i].z, num[4 * i + 2]);
        num[4 * i + 3] = fmaf(f, o[k][i].w, num[4 * i + 3]);
      }
    }
  }
  const float inv = den > 0.f ? 1.f / den : 0.f;
  const int tok = tok0 + r / n_rep, h = g * n_rep + r % n_rep;
  uint32_t w[JOIN / 2];
#pragma unroll
  for (int i = 0; i < JOIN / 2; ++i) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(num[2 * i] * inv, num[2 * i + 1] * inv);
    w[i] = *(const uint32_t*)&x;
  }
  uint4* dst = (uint4*)(out + (size_t)tok * out_stride + (size_t)h * HD + part * JOIN);
#pragma unroll
  for (int i = 0; i < JOIN / 8; ++i) dst[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  if (lse && part == 0) lse[(size_t)tok * nh + h] = lost ? INFINITY : m + log2f(den);
}

template <int HD, int NT, int MODE = PF_PLAIN>
static int launch_ws(const void* q, int q_stride, void* out, int out_stride, const void* k_pages, const void* v_pages,
                     int n_pages, const int* page_table, int table_width, const int* cu_seqlens, const int* ctx_lens,
                     int B, int max_new, int nh, int nkv, float scale, int window, int* status, cudaStream_t stream,
                     int sinks = 0, float* lse = nullptr, int n_splits = 1, float* part = nullptr) {
  using W = WsCfg<HD, NT>;
  static int configured[MAX_DEVICES];
  if (int rc = allow_smem(prefill_ws_kernel<HD, NT, MODE>, W::SMEM, configured)) return rc;
  // the cache as a matrix [n_pages * nkv * PAGE, HD]: a page of one KV head is 64 of its rows
  const long rows = (long)n_pages * nkv * PAGE;
  if (rows > 0x7fffffffL) return WPC_ERR_TOO_LARGE;
  CUtensorMap mk, mv;
  int rc = tc::tensor_map(k_pages, (int)rows, HD, HD, PAGE, &mk);
  if (rc) return rc;
  rc = tc::tensor_map(v_pages, (int)rows, HD, HD, PAGE, &mv);
  if (rc) return rc;
  const int n_rep = nh / nkv;
  dim3 grid(nkv, (max_new * n_rep + NT * ROWS - 1) / (NT * ROWS), B * n_splits);
  float4* part_o = (float4*)part;
  float2* part_ml = (float2*)(part_o + (size_t)grid.x * grid.y * grid.z * ROWS * (HD / 4));
  wpc::launch(prefill_ws_kernel<HD, NT, MODE>, grid, W::THREADS, W::SMEM, stream, mk, mv, (const __nv_bfloat16*)q, q_stride,
              (__nv_bfloat16*)out, out_stride, page_table, table_width, cu_seqlens, ctx_lens, nh, nkv, scale * LOG2E,
              window, status, wait_policy().limit_ns, wait_policy().starve, NT == 1 ? sm_count() : 1 << 30,
              max_new >= 1024 ? 1 : 0, sinks, lse, n_splits, part_o, part_ml);
  if constexpr ((MODE & PF_SHARED) != 0) {
    if (int e = launch_status()) return e;
    grid.z = B * (HD / JOIN);
    wpc::launch(prefill_join_kernel<HD>, grid, ROWS, 0, stream, part_o, part_ml, (__nv_bfloat16*)out, out_stride, lse,
                cu_seqlens, nh, nkv, n_splits);
  }
  return launch_status();
}

}  // namespace fatc
}  // namespace wpc

extern "C" {

int wpc_attention_prefill_tc_supports(int nh, int nkv, int hd) {
  return (hd == 64 || hd == 128) && nkv >= 1 && nh % nkv == 0 && nh / nkv <= 128;
}

// tiles: 1 or 2 row tiles of 128 rows to a CTA (1: two CTAs to an SM, the faster one: 54 against
// 60 us at 2,048 tokens of the 7B shape, 480 against 659 us at 8,192).  n_pages: pages of the cache.
// q rows and out rows must be 16-byte aligned (strides multiples of 8 elements).
int wpc_attention_prefill_tc(const void* q, int q_stride, void* out, int out_stride, const void* k_pages,
                             const void* v_pages, const int* page_table, int table_width, const int* cu_seqlens,
                             const int* ctx_lens, int B, int max_new, int nh, int nkv, int hd, float scale,
                             int window, int* status, int n_pages, int tiles, cudaStream_t stream) {
  if (B <= 0 || max_new <= 0) return 0;
  if (!wpc_attention_prefill_tc_supports(nh, nkv, hd) || (q_stride % 8) || (out_stride % 8) ||
      (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15))
    return WPC_ERR_UNSUPPORTED;
  if (tiles == 1 || tiles == 2) {
    // one or two row tiles to a CTA
#define WPC_WS(HD_, NT_)                                                                                          \
  return wpc::fatc::launch_ws<HD_, NT_>(q, q_stride, out, out_stride, k_pages, v_pages, n_pages, page_table,      \
                                        table_width, cu_seqlens, ctx_lens, B, max_new, nh, nkv, scale, window,     \
                                        status, stream)
    if (hd == 128 && tiles == 2) WPC_WS(128, 2);
    if (hd == 128) WPC_WS(128, 1);
    if (tiles == 2) WPC_WS(64, 2);
    WPC_WS(64, 1);
#undef WPC_WS
  }
  return WPC_ERR_BAD_ARGUMENT;
}

// The same with sinks beside a window, and, where lse is given (no window, no sinks), each row's
// maximum + log2(sum) into lse [T][nh].  One row tile to a CTA, or, with n_splits > 1, that many CTAs to a
// tile, joined by a second kernel; part: float32 [n_splits * tiles * 128 * (hd + 2)], 16-byte aligned, tiles being
// ceil(max_new * nh / nkv / 128) * nkv * B.
int wpc_attention_prefill_tc_bounded(const void* q, int q_stride, void* out, int out_stride, const void* k_pages,
                                     const void* v_pages, const int* page_table, int table_width,
                                     const int* cu_seqlens, const int* ctx_lens, int B, int max_new, int nh, int nkv,
                                     int hd, float scale, int window, int sinks, float* lse, int* status, int n_pages,
                                     int n_splits, float* part, cudaStream_t stream) {
  if (B <= 0 || max_new <= 0) return 0;
  if (!wpc_attention_prefill_tc_supports(nh, nkv, hd) || (q_stride % 8) || (out_stride % 8) ||
      (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15))
    return WPC_ERR_UNSUPPORTED;
  if (lse ? (window > 0 || sinks != 0) : (sinks < 1 || window < 1)) return WPC_ERR_BAD_ARGUMENT;
  if (n_splits < 1 || n_splits > 64 || (n_splits > 1 && (!part || ((uintptr_t)part & 15) || (long)B * n_splits > 65535 || B > 8191)))
    return WPC_ERR_BAD_ARGUMENT;
#define WPC_WS(HD_, MODE_)                                                                                           \
  return wpc::fatc::launch_ws<HD_, 1, MODE_>(q, q_stride, out, out_stride, k_pages, v_pages, n_pages, page_table,  \
                                              table_width, cu_seqlens, ctx_lens, B, max_new, nh, nkv, scale, window, \
                                              status, stream, sinks, lse, n_splits, part)
  using namespace wpc::fatc;
#define WPC_FORMS(HD_)                                        \
  if (n_splits > 1 && sinks) WPC_WS(HD_, PF_SINKS | PF_SHARED); \
  if (n_splits > 1) WPC_WS(HD_, PF_SUMS | PF_SHARED);           \
  if (sinks) WPC_WS(HD_, PF_SINKS);                             \
  WPC_WS(HD_, PF_SUMS)
  if (hd == 128) {
    WPC_FORMS(128);
  }
  WPC_FORMS(64);
#undef WPC_FORMS
#undef WPC_WS
}

}  // extern "C"
