// What stays in a cache of bounded size, and its move together.
//
// select_kept: of the n entries that a sequence holds for a KV head, `keep` stay: those of its first
// `sinks` positions, those of its last `recent` positions, and of the others the ones that attention
// gave the most weight (weight_sums, see attention_sums.cu), ties to the entry stored first.  An
// entry is ranked by a 32-bit key: all ones if it is protected, else its sum's bits turned
// into an unsigned number of the same order (a NaN counts as -inf).  The keep-th greatest key is
// found digit by digit, by counting.
//
// An entry that stays and is stored below `keep` does not move; the others that stay, all behind,
// fill the holes in order.  So what moves is as little as can be, sources and targets never
// overlap, and all moves can run at once.
//
// move_kept: the moves: keys, values, sums and positions.
//
// Measured (4 KV heads of 128): the choice of 2,048 of up to 4,096 entries, 28 layers and 8 sequences, 13.0 us (25 MB,
// 3.8 us at the copy's rate; bound by the counting in shared memory), 44 with the keys read again for each of
// four digits; one layer of 1,088 entries 4.6, latency; beyond 32,768 entries 207 us for 20,000 of 40,000, 28 layers,
// and 312 for 55,000 of 60,000 (loads one behind the other, by one block a row).  The moves that follow, 471 MB, 86 us, 5.5 TB/s on rows of
// 256 bytes (159 with one row on its way at a time).
#include "api.h"
#include "common.cuh"

namespace wpc {

constexpr uint32_t SEL_PROTECTED = 0xffffffffu;

__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);          // (-0 becomes +0)
  return u & 0x80000000u ? ~u : u | 0x80000000u;        // at most 0xff800000, for +inf
}

// Where the entries of a (layer, sequence, KV head) are, and their keys.
struct Entries {
  const float* sums;               // of the layer
  const int* positions;
  const int* table;                // of the sequence
  int nkv, g, n_pages, sinks, first_recent;
  __device__ __forceinline__ uint32_t key_of(float w, int p) const {
    return p < sinks || p >= first_recent ? SEL_PROTECTED : order_key(w);
  }
  // place of entry i in the records, -1 without a page
  __device__ __forceinline__ long at(int i) const {
    const int page = table[i / WPC_PAGE];
    return page < 0 || page >= n_pages ? -1 : ((long)page * nkv + g) * WPC_PAGE + i % WPC_PAGE;
  }
};

// Exclusive sum of `v` over the block's NT threads; *total: the sum of all.  red: 32 ints of this
// call's own (two arrays in turn do for any number of calls: each has a barrier inside).
template <int NT>
__device__ __forceinline__ int block_scan(int v, int* red, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  if (lane == 31) red[warp] = incl;
  __syncthreads();
  int w = lane < NT / 32 ? red[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += t;
  }
  *total = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
  return (warp ? before : 0) + incl - v;
}

// ---- up to NT * ITEMS entries: their keys stay in registers ------------------------------------------
// A block to a (layer, sequence, KV head); a thread owns ITEMS consecutive entries, which lie in one
// page.  The keep-th greatest key is found in three digits of 11, 11 and 10 bits by histograms in
// shared memory (with 8-bit digits the first one holds hardly more than the exponent, and
// nearly all additions of a block would meet in a few bins); a digit whose bin is wanted whole
// ends the search.  Then two scans give ties, holes and movers their ranks.
template <int NT, int ITEMS>
__global__ void __launch_bounds__(NT)
select_kept_kernel(const float* weight_sums, const int* stored_positions, size_t layer_stride,
                   const int* __restrict__ page_table, int table_width, const int* __restrict__ lens,
                   const int* __restrict__ next_positions, int nkv, int n_pages, int keep, int sinks, int recent,
                   int* kept, int* status) {
  constexpr int BINS = 2048, PER = BINS / NT;
  pdl_trigger();
  extern __shared__ int smem[];
  int* const places = smem;                             // [keep] what belongs at each place
  int* const holes = smem + keep;                       // [keep]
  __shared__ __align__(16) int hist[BINS];
  __shared__ int red[2][32];
  __shared__ int s_digit, s_want, s_count;
  const int g = blockIdx.x, b = blockIdx.y, layer = blockIdx.z, B = gridDim.y, tid = threadIdx.x;
  for (int i = tid; i < BINS; i += NT) hist[i] = 0;
  pdl_wait();
  int* const out = kept + (((size_t)layer * B + b) * nkv + g) * keep;
  const int n = min(max(lens[b], 0), table_width * WPC_PAGE);
  if (n <= keep) {                                      // nothing has to go
    for (int i = tid; i < keep; i += NT) out[i] = i < n ? i : -1;
    return;
  }
  const Entries e{weight_sums + layer * layer_stride, stored_positions + layer * layer_stride,
                  page_table + (size_t)b * table_width, nkv, g, n_pages, sinks, next_positions[b] - recent};
  const int i0 = tid * ITEMS;
  uint32_t key[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) key[j] = 0;
  if (i0 < n) {
    const long at = e.at(i0);
    if (at < 0) {
      if (status) atomicExch(status, WPC_ERR_BAD_ARGUMENT);
    } else {
#pragma unroll
      for (int j = 0; j < ITEMS; j += 4) {
        const float4 w = *(const float4*)(e.sums + at + j);
        const int4 p = *(const int4*)(e.positions + at + j);
        key[j] = e.key_of(w.x, p.x);
        key[j + 1] = e.key_of(w.y, p.y);
        key[j + 2] = e.key_of(w.z, p.z);
        key[j + 3] = e.key_of(w.w, p.w);
      }
    }
  }
  const int mine = min(max(n - i0, 0), ITEMS);          // entries that exist
  uint32_t prefix = 0, mask = 0;
  int want = keep, which = 0;
  __syncthreads();                                      // hist is zero
#pragma unroll
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
    const uint32_t bins = digit == 2 ? 1023u : 2047u;
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (j < mine && (key[j] & mask) == prefix) atomicAdd(&hist[(key[j] >> shift) & bins], 1);
    __syncthreads();
    int c[PER], sum = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {                     // the highest bins belong to the first thread
      c[j] = hist[BINS - 1 - tid * PER - j];
      hist[BINS - 1 - tid * PER - j] = 0;               // for the next digit
      sum += c[j];
    }
    int total;
    int above = block_scan<NT>(sum, red[which], &total);
    which ^= 1;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (above < want && above + c[j] >= want) {
        s_digit = BINS - 1 - tid * PER - j;
        s_want = want - above;
        s_count = c[j];
      }
      above += c[j];
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit << shift;
    mask |= bins << shift;
    want = s_want;
    if (s_count == want) break;                         // the bin is wanted whole
    __syncthreads();                                    // (s_digit and its like are written again)
  }
  const bool some_ties = s_count != want;

  // ---- an entry stays if its digits are greater, or equal and it is among the first `want` of those ----
  int total, rank = 0;
  if (some_ties) {
    int ties = 0;
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) ties += j < mine && (key[j] & mask) == prefix;
    rank = block_scan<NT>(ties, red[which], &total);
    which ^= 1;
  }
  uint32_t stays = 0;
  int n_holes = 0, n_movers = 0;
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const uint32_t k = key[j] & mask;
    const bool tie = j < mine && k == prefix;
    const bool stay = (j < mine && k > prefix) || (tie && (!some_ties || rank < want));
    rank += tie;
    stays |= (stay ? 1u : 0u) << j;
    n_holes += !stay && i0 + j < keep;                  // (n > keep: every place below keep has an entry)
    n_movers += stay && i0 + j >= keep;
  }
  const int ranks = block_scan<NT>(n_holes | n_movers << 16, red[which], &total);   // both at most 32,767
  int hole = ranks & 0xffff, mover = ranks >> 16;
#pragma unroll
  for (int j = 0; j < ITEMS; ++j)
    if (i0 + j < keep) {
      if (stays >> j & 1) places[i0 + j] = i0 + j;
      else holes[hole++] = i0 + j;
    }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ITEMS; ++j)
    if (i0 + j >= keep && (stays >> j & 1)) places[holes[mover++]] = i0 + j;
  __syncthreads();
  for (int i = tid; i < keep; i += NT) out[i] = places[i];
}

// ---- any number of entries ----------------------------------------------------------------------------
// The same with the keys made anew from the records each time, eight bits a digit.  The list of holes lies
// in shared memory, or, where it has no room there, in `scratch`, [rows][keep].
constexpr int SEL_THREADS = 1024;

__global__ void __launch_bounds__(SEL_THREADS)
select_kept_long_kernel(const float* weight_sums, const int* stored_positions, size_t layer_stride,
                        const int* __restrict__ page_table, int table_width, const int* __restrict__ lens,
                        const int* __restrict__ next_positions, int nkv, int n_pages, int keep, int sinks, int recent,
                        int* kept, int* scratch, int* status) {
  pdl_trigger();
  pdl_wait();
  extern __shared__ int smem[];
  __shared__ int hist[256];
  __shared__ int red[2][32];
  __shared__ uint32_t s_digit;
  __shared__ int s_want;
  const int g = blockIdx.x, b = blockIdx.y, layer = blockIdx.z, B = gridDim.y, tid = threadIdx.x;
  const size_t row = ((size_t)layer * B + b) * nkv + g;
  int* const out = kept + row * keep;
  int* const holes = scratch ? scratch + row * keep : smem;             // [keep]
  const int n = min(max(lens[b], 0), table_width * WPC_PAGE);
  if (n <= keep) {
    for (int i = tid; i < keep; i += SEL_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  const Entries e{weight_sums + layer * layer_stride, stored_positions + layer * layer_stride,
                  page_table + (size_t)b * table_width, nkv, g, n_pages, sinks, next_positions[b] - recent};
  bool bad = false;
  auto key = [&](int i) -> uint32_t {
    const long at = e.at(i);
    bad = bad || at < 0;
    return at < 0 ? 0u : e.key_of(e.sums[at], e.positions[at]);
  };
  uint32_t prefix = 0;
  int want = keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    for (int i = tid; i < n; i += SEL_THREADS) {
      const uint32_t k = key(i);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid < 32) {
      // lane l holds the eight bins 255 - 8 l .. downwards; how many lie above each
      int c[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) { c[j] = hist[255 - 8 * tid - j]; sum += c[j]; }
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, o);
        if (tid >= o) incl += t;
      }
      int above = incl - sum;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (above < want && above + c[j] >= want) {
          s_digit = (uint32_t)(255 - 8 * tid - j);
          s_want = want - above;
        }
        above += c[j];
      }
    }
    __syncthreads();
    prefix |= s_digit << shift;
    want = s_want;
  }
  int ties = 0, n_holes = 0, n_movers = 0, which = 0;   // of all entries before this round's
  for (int i0 = 0; i0 < n; i0 += SEL_THREADS) {
    const int i = i0 + tid;
    const uint32_t k = i < n ? key(i) : 0u;
    const bool tie = i < n && k == prefix;
    int total;
    const int rank = ties + block_scan<SEL_THREADS>(tie ? 1 : 0, red[which], &total);
    which ^= 1;
    ties += total;
    const bool stays = i < n && (k > prefix || (tie && rank < want));
    const bool hole = i < keep && !stays, mover = i >= keep && stays;
    const int at = block_scan<SEL_THREADS>((hole ? 1 : 0) | (mover ? 1 << 16 : 0), red[which], &total);
    which ^= 1;
    if (i < keep && stays) out[i] = i;
    if (hole) holes[n_holes + (at & 0xffff)] = i;
    n_holes += total & 0xffff;
    // (holes lie below keep, movers from keep on: a mover's hole was found in an earlier round or
    // in this one)
    __syncthreads();
    if (mover) out[holes[n_movers + (at >> 16)]] = i;
    n_movers += total >> 16;
  }
  if (bad && status) atomicExch(status, WPC_ERR_BAD_ARGUMENT);
}

// ---- the moves --------------------------------------------------------------------------------------------
// A block to MOVE_PLACES places of the kept part of a (layer, sequence, KV head): it lists the moves among
// them in shared memory, then its threads copy the listed rows, chunk by chunk, several loads
// each before the first store (a row at a time would be a trip to memory for every row).
constexpr int MOVE_THREADS = 256, MOVE_PLACES = 256, MOVE_DEPTH = 4;

template <typename V>
__global__ void __launch_bounds__(MOVE_THREADS)
move_kept_kernel(V* k_pages, V* v_pages, int k_chunks, int v_chunks, float* weight_sums, int* stored_positions,
                 const int* __restrict__ page_table, int table_width, const int* kept, int B, int nkv, int n_pages,
                 int keep, int* status) {
  // (no early start of the kernel behind: decode attention reads pages of earlier positions ahead of its
  // dependency wait, which is right only if nothing on the stream still writes them)
  __shared__ long s_from[MOVE_PLACES], s_to[MOVE_PLACES];
  __shared__ int s_n;
  if (threadIdx.x == 0) s_n = 0;
  pdl_wait();
  const int g = blockIdx.x % nkv, b = blockIdx.x / nkv, layer = blockIdx.z, tid = threadIdx.x, lane = tid & 31;
  const int i = blockIdx.y * MOVE_PLACES + tid;
  const int* table = page_table + (size_t)b * table_width;
  const int src = i < keep ? kept[(((size_t)layer * B + b) * nkv + g) * keep + i] : -1;
  long from = 0, to = 0;
  bool moves = src >= 0 && src != i;
  if (moves) {
    const int sb = src / WPC_PAGE, db = i / WPC_PAGE;
    const int sp = sb < table_width ? table[sb] : -1, dp = db < table_width ? table[db] : -1;
    if (src < keep || sp < 0 || sp >= n_pages || dp < 0 || dp >= n_pages) {
      moves = false;
      if (status) atomicExch(status, WPC_ERR_BAD_ARGUMENT);
    } else {
      from = (((long)layer * n_pages + sp) * nkv + g) * WPC_PAGE + src % WPC_PAGE;
      to = (((long)layer * n_pages + dp) * nkv + g) * WPC_PAGE + i % WPC_PAGE;
    }
  }
  __syncthreads();
  const uint32_t who = __ballot_sync(0xffffffffu, moves);
  int first = 0;
  if (lane == 0 && who) first = atomicAdd(&s_n, __popc(who));               // (the order of the moves does not matter)
  first = __shfl_sync(0xffffffffu, first, 0);
  if (moves) {
    const int at = first + __popc(who & ((1u << lane) - 1));
    s_from[at] = from;
    s_to[at] = to;
    weight_sums[to] = weight_sums[from];
    stored_positions[to] = stored_positions[from];
  }
  __syncthreads();
  const int chunks = k_chunks + v_chunks, all = s_n * chunks;
  for (int c0 = tid; c0 < all; c0 += MOVE_THREADS * MOVE_DEPTH) {
    V v[MOVE_DEPTH];
    V* dst[MOVE_DEPTH];
#pragma unroll
    for (int j = 0; j < MOVE_DEPTH; ++j) {
      const int c = c0 + j * MOVE_THREADS;
      dst[j] = nullptr;
      if (c < all) {
        const int m = c / chunks, in = c - m * chunks;
        const bool key = in < k_chunks;
        const V* from_p = key ? k_pages + s_from[m] * k_chunks + in : v_pages + s_from[m] * v_chunks + (in - k_chunks);
        dst[j] = key ? k_pages + s_to[m] * k_chunks + in : v_pages + s_to[m] * v_chunks + (in - k_chunks);
        v[j] = *from_p;
      }
    }
#pragma unroll
    for (int j = 0; j < MOVE_DEPTH; ++j)
      if (dst[j]) *dst[j] = v[j];
  }
}

}  // namespace wpc

using namespace wpc;

// Places that the kernels keep in shared memory for every (layer, sequence, KV head); a table that holds
// no more entries than are kept loses nothing.
static int kept_places(int keep, int table_width) { return keep < (long)table_width * WPC_PAGE ? keep : 0; }
constexpr int SEL_MAX_SHARED = 50 * 1024;

extern "C" {

long wpc_select_kept_scratch(int keep, int table_width) {
  const int places = kept_places(keep, table_width);
  return places > SEL_MAX_SHARED ? places : 0;
}

int wpc_select_kept(const float* weight_sums, const int* stored_positions, const int* page_table, int table_width,
                    const int* lens, const int* next_positions, int layers, int B, int nkv, int n_pages,
                    int keep, int sinks, int recent, int* kept, int* scratch, int* status, cudaStream_t stream) {
  if (layers <= 0 || B <= 0 || nkv <= 0) return 0;
  if (keep < 1 || sinks < 0 || recent < 0 || sinks > keep - recent || n_pages < 1 || table_width < 0) return WPC_ERR_BAD_ARGUMENT;
  if (layers > 65535 || B > 65535) return WPC_ERR_UNSUPPORTED;
  const long n = (long)table_width * WPC_PAGE;
  const int places = kept_places(keep, table_width);
  const bool far = wpc_select_kept_scratch(keep, table_width) > 0;
  if (far && !scratch) return WPC_ERR_BAD_ARGUMENT;
  const bool wide = (((uintptr_t)weight_sums | (uintptr_t)stored_positions) & 15) == 0;
  const dim3 grid(nkv, B, layers);
  const size_t layer_stride = (size_t)n_pages * nkv * WPC_PAGE;
  // A thread's share of the keys stays in registers as long as a block of 1,024 threads holds them all
  // (and the records can be read 16 bytes a load): 32,768 entries, 16,384 of which stay, 28 layers 34.6 us, 165
  // read again for each digit.  Few keys a thread where they fit: 8,192 entries 12.2 us with eight,
  // 19.2 with thirty-two; 4,096 entries 6.6 with 512 threads, 10.0 with 1,024 (8 sequences: 20.2 and 33.7).
#define WPC_SELECT(NT, ITEMS)                                                                                        \
  do {                                                                                                               \
    static int configured[MAX_DEVICES];                                                                              \
    if (int rc = allow_smem(select_kept_kernel<NT, ITEMS>, places * 8, configured)) return rc;                       \
    wpc::launch(select_kept_kernel<NT, ITEMS>, grid, NT, places * 8, stream, weight_sums, stored_positions,          \
                layer_stride, page_table, table_width, lens, next_positions, nkv, n_pages, keep, sinks, recent, kept, \
                status);                                                                                             \
  } while (0)
  if (wide && n <= 512 * 8) WPC_SELECT(512, 8);
  else if (wide && n <= 1024 * 8) WPC_SELECT(1024, 8);
  else if (wide && n <= 1024 * 32 && places <= 24 * 1024) WPC_SELECT(1024, 32);
  else {
    static int configured[MAX_DEVICES];
    const int smem = far ? 0 : places * 4;
    if (int rc = allow_smem(select_kept_long_kernel, smem, configured)) return rc;
    wpc::launch(select_kept_long_kernel, grid, SEL_THREADS, smem, stream, weight_sums, stored_positions, layer_stride,
                page_table, table_width, lens, next_positions, nkv, n_pages, keep, sinks, recent, kept,
                far ? scratch : nullptr, status);
  }
#undef WPC_SELECT
  return launch_status();
}

int wpc_move_kept(void* k_pages, void* v_pages, int k_bytes, int v_bytes, float* weight_sums, int* stored_positions,
                  const int* page_table, int table_width, const int* kept, int layers, int B, int nkv, int n_pages,
                  int keep, int* status, cudaStream_t stream) {
  if (layers <= 0 || B <= 0 || nkv <= 0 || keep <= 0) return 0;
  const int chunks = (keep - 1) / MOVE_PLACES + 1;
  if (layers > 65535 || (long)B * nkv > 0x7fffffffL || chunks > 65535) return WPC_ERR_TOO_LARGE;
  const dim3 grid((unsigned)(B * nkv), (unsigned)chunks, (unsigned)layers);
  const uintptr_t align = (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)k_bytes | (uintptr_t)v_bytes;
  auto go = [&](auto kernel, auto* k, auto* v) {
    wpc::launch(kernel, grid, MOVE_THREADS, 0, stream, k, v, k_bytes / (int)sizeof(*k), v_bytes / (int)sizeof(*v), weight_sums,
                stored_positions, page_table, table_width, kept, B, nkv, n_pages, keep, status);
  };
  if (align % 16 == 0) go(move_kept_kernel<uint4>, (uint4*)k_pages, (uint4*)v_pages);
  else if (align % 4 == 0) go(move_kept_kernel<uint32_t>, (uint32_t*)k_pages, (uint32_t*)v_pages);
  else if (align % 2 == 0) go(move_kept_kernel<uint16_t>, (uint16_t*)k_pages, (uint16_t*)v_pages);
  else return WPC_ERR_UNSUPPORTED;
  PdlWaiting::all().add(stream);      // (the kernel behind starts when the moves are done and visible)
  return launch_status();
}

}  // extern "C"
