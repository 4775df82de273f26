// Where the sums of attention weights go (attention_sums.cu, attention_sums_tc.cu).
#pragma once
#include "common.cuh"

namespace wpc {

struct SumsTarget {
  const int* page_table;
  int table_width, n_pages;
  const int* token_positions;       // [T]
  float* weight_sums;               // [n_pages, nkv, PAGE]
  int* stored_positions;            // [n_pages, nkv, PAGE]
  int* status;
};

// The kernels' grids go by the longest length that the caller stated: a sequence beyond what they cover
// (`covered` keys) is an error that the host learns of.  For one thread of the sequence.
__device__ __forceinline__ void check_length(const SumsTarget& t, int length, int covered) {
  if (length > covered && t.status) atomicExch(t.status, WPC_ERR_BAD_ARGUMENT);
}

// Adds the sum `w` of key `key` of (sequence b, KV head g); token: the step's token that wrote this
// key, -1 for a key of an earlier step.
__device__ __forceinline__ void add_sum(const SumsTarget& t, int nkv, int b, int g, int key, int token, float w) {
  const int block = key / WPC_PAGE;
  const int page = block < t.table_width ? t.page_table[(size_t)b * t.table_width + block] : -1;
  if (page < 0 || page >= t.n_pages) {
    if (t.status) atomicExch(t.status, WPC_ERR_BAD_ARGUMENT);
    return;
  }
  const size_t at = ((size_t)page * nkv + g) * WPC_PAGE + key % WPC_PAGE;
  t.weight_sums[at] = token >= 0 ? w : t.weight_sums[at] + w;
  if (token >= 0) t.stored_positions[at] = t.token_positions[token];
}

}  // namespace wpc
