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
#include "api.h"
#include "common.cuh"

namespace wpc {

constexpr int SEL_THREADS = 512;
constexpr uint32_t SEL_PROTECTED = 0xffffffffu;

__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);          // (-0 becomes +0)
  return u & 0x80000000u ? ~u : u | 0x80000000u;        // at most 0xff800000, for +inf
}

// Exclusive sum over the block's threads of `v`; *total: the sum of all.  red: 17 ints.
__device__ __forceinline__ int block_scan(int v, int* red, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  __syncthreads();
  if (lane == 31) red[warp] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < SEL_THREADS / 32; ++i) {
    const int x = red[i];
    before += i < warp ? x : 0;
    all += x;
  }
  *total = all;
  return before + incl - v;
}

// A block to a (layer, sequence, KV head).  Shared memory: the holes' places (keep ints), and
// with KEYS the keys of all entries (else they are made again from memory each time).
template <bool KEYS>
__global__ void __launch_bounds__(SEL_THREADS)
select_kept_kernel(const float* __restrict__ weight_sums, const int* __restrict__ stored_positions, size_t layer_stride,
                   const int* __restrict__ page_table, int table_width, const int* __restrict__ lens,
                   const int* __restrict__ next_positions, int nkv, int n_pages, int keep, int sinks, int recent,
                   int* __restrict__ kept, int* __restrict__ status) {
  pdl_trigger();
  pdl_wait();
  extern __shared__ uint32_t smem[];
  int* holes = (int*)smem;                              // [keep]
  uint32_t* keys = smem + keep;                         // [n]
  __shared__ int hist[256];
  __shared__ int red[SEL_THREADS / 32];
  __shared__ uint32_t s_digit;
  __shared__ int s_want;
  const int g = blockIdx.x, b = blockIdx.y, layer = blockIdx.z, B = gridDim.y, tid = threadIdx.x;
  int* out = kept + (((size_t)layer * B + b) * nkv + g) * keep;
  const int* table = page_table + (size_t)b * table_width;
  const int n = min(max(lens[b], 0), table_width * WPC_PAGE);
  if (n <= keep) {                                      // nothing has to go
    for (int i = tid; i < keep; i += SEL_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  const int first_recent = next_positions[b] - recent;
  bool bad = false;
  auto key_of = [&](int i) -> uint32_t {
    const int page = table[i / WPC_PAGE];
    if (page < 0 || page >= n_pages) { bad = true; return 0u; }
    const size_t at = layer * layer_stride + ((size_t)page * nkv + g) * WPC_PAGE + i % WPC_PAGE;
    const int p = stored_positions[at];
    return (p < sinks || p >= first_recent) ? SEL_PROTECTED : order_key(weight_sums[at]);
  };
  if (KEYS) {
    for (int i = tid; i < n; i += SEL_THREADS) keys[i] = key_of(i);
  }
  auto key = [&](int i) { return KEYS ? keys[i] : key_of(i); };

  // ---- the keep-th greatest key, eight bits at a time; `want`: how many of those that share
  // the digits found so far are still to be taken ----
  uint32_t prefix = 0;
  int want = keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = tid; i < 256; i += SEL_THREADS) hist[i] = 0;
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

  // ---- every entry: kept if its key is greater, or equal and among the first `want` of those ----
  int ties = 0, n_holes = 0, n_movers = 0;              // of all entries before this round's
  for (int i0 = 0; i0 < n; i0 += SEL_THREADS) {
    const int i = i0 + tid;
    const uint32_t k = i < n ? key(i) : 0u;
    const bool tie = i < n && k == prefix;
    int total;
    const int rank = ties + block_scan(tie ? 1 : 0, red, &total);
    ties += total;
    const bool stays = i < n && (k > prefix || (tie && rank < want));
    const bool hole = i < keep && !stays, mover = i >= keep && stays;
    const int at = block_scan((hole ? 1 : 0) | (mover ? 1 << 16 : 0), red, &total);
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

constexpr int MOVE_THREADS = 256;

// A warp to 32 places of the kept part of a (layer, sequence, KV head).
template <typename V>
__global__ void __launch_bounds__(MOVE_THREADS)
move_kept_kernel(uint8_t* __restrict__ k_pages, uint8_t* __restrict__ v_pages, int k_bytes, int v_bytes,
                 float* __restrict__ weight_sums, int* __restrict__ stored_positions, const int* __restrict__ page_table,
                 int table_width, const int* __restrict__ kept, int B, int nkv, int n_pages, int keep,
                 int* __restrict__ status) {
  // (no early start of the kernel behind: decode attention reads pages of earlier positions ahead of its
  // dependency wait, which is right only if nothing on the stream still writes them)
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.y;                           // (layer, sequence, KV head)
  const int g = row % nkv, b = (row / nkv) % B, layer = row / (nkv * B);
  const int i = (blockIdx.x * (MOVE_THREADS / 32) + warp) * 32 + lane;
  const int* table = page_table + (size_t)b * table_width;
  const int src = i < keep ? kept[(size_t)row * keep + i] : -1;
  size_t from = 0, to = 0;
  bool moves = src >= 0 && src != i;
  if (moves) {
    const int sb = src / WPC_PAGE, db = i / WPC_PAGE;
    const int sp = sb < table_width ? table[sb] : -1, dp = db < table_width ? table[db] : -1;
    if (src < keep || sp < 0 || sp >= n_pages || dp < 0 || dp >= n_pages) {
      moves = false;
      if (status) atomicExch(status, WPC_ERR_BAD_ARGUMENT);
    } else {
      from = (((size_t)layer * n_pages + sp) * nkv + g) * WPC_PAGE + src % WPC_PAGE;
      to = (((size_t)layer * n_pages + dp) * nkv + g) * WPC_PAGE + i % WPC_PAGE;
      weight_sums[to] = weight_sums[from];
      stored_positions[to] = stored_positions[from];
    }
  }
  for (uint32_t left = __ballot_sync(0xffffffffu, moves); left; left &= left - 1) {
    const int l = __ffs(left) - 1;
    const size_t f = __shfl_sync(0xffffffffu, from, l), t = __shfl_sync(0xffffffffu, to, l);
    for (int e = lane * (int)sizeof(V); e < k_bytes; e += 32 * (int)sizeof(V))
      *(V*)(k_pages + t * k_bytes + e) = *(const V*)(k_pages + f * k_bytes + e);
    for (int e = lane * (int)sizeof(V); e < v_bytes; e += 32 * (int)sizeof(V))
      *(V*)(v_pages + t * v_bytes + e) = *(const V*)(v_pages + f * v_bytes + e);
  }
}

}  // namespace wpc

using namespace wpc;

extern "C" {

int wpc_select_kept(const float* weight_sums, const int* stored_positions, const int* page_table, int table_width,
                    const int* lens, const int* next_positions, int layers, int B, int nkv, int n_pages,
                    int keep, int sinks, int recent, int* kept, int* status, cudaStream_t stream) {
  if (layers <= 0 || B <= 0 || nkv <= 0) return 0;
  if (keep < 1 || sinks < 0 || recent < 0 || sinks > keep - recent || n_pages < 1 || table_width < 0) return WPC_ERR_BAD_ARGUMENT;
  if (layers > 65535 || B > 65535) return WPC_ERR_UNSUPPORTED;
  const long holes = (long)keep * 4, keys = (long)table_width * WPC_PAGE * 4, most = 200 * 1024;
  if (holes > most) return WPC_ERR_TOO_LARGE;
  const dim3 grid(nkv, B, layers);
  const size_t layer_stride = (size_t)n_pages * nkv * WPC_PAGE;
  if (holes + keys <= most) {
    static int configured[MAX_DEVICES];
    if (int rc = allow_smem(select_kept_kernel<true>, (int)(holes + keys), configured)) return rc;
    wpc::launch(select_kept_kernel<true>, grid, SEL_THREADS, holes + keys, stream, weight_sums, stored_positions, layer_stride,
                page_table, table_width, lens, next_positions, nkv, n_pages, keep, sinks, recent, kept, status);
  } else {
    static int configured[MAX_DEVICES];
    if (int rc = allow_smem(select_kept_kernel<false>, (int)holes, configured)) return rc;
    wpc::launch(select_kept_kernel<false>, grid, SEL_THREADS, holes, stream, weight_sums, stored_positions, layer_stride,
                page_table, table_width, lens, next_positions, nkv, n_pages, keep, sinks, recent, kept, status);
  }
  return launch_status();
}

int wpc_move_kept(void* k_pages, void* v_pages, int k_bytes, int v_bytes, float* weight_sums, int* stored_positions,
                  const int* page_table, int table_width, const int* kept, int layers, int B, int nkv, int n_pages,
                  int keep, int* status, cudaStream_t stream) {
  if (layers <= 0 || B <= 0 || nkv <= 0 || keep <= 0) return 0;
  const long rows = (long)layers * B * nkv;
  if (rows > 65535) return WPC_ERR_TOO_LARGE;
  const dim3 grid((keep + MOVE_THREADS - 1) / MOVE_THREADS, (unsigned)rows);
  const uintptr_t align = (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)k_bytes | (uintptr_t)v_bytes;
  auto go = [&](auto kernel) {
    wpc::launch(kernel, grid, MOVE_THREADS, 0, stream, (uint8_t*)k_pages, (uint8_t*)v_pages, k_bytes, v_bytes, weight_sums,
                stored_positions, page_table, table_width, kept, B, nkv, n_pages, keep, status);
  };
  if (align % 16 == 0) go(move_kept_kernel<uint4>);
  else if (align % 4 == 0) go(move_kept_kernel<uint32_t>);
  else if (align % 2 == 0) go(move_kept_kernel<uint16_t>);
  else return WPC_ERR_UNSUPPORTED;
  pdl_skip_next() = 1;      // (the kernel behind starts when the moves are done and visible)
  return launch_status();
}

}  // extern "C"
