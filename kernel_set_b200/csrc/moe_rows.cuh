// What the forward and the backward steps of a routed layer share: the checks of a pair count and the map from
// pairs to sorted rows.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "common.cuh"

namespace ksb {

constexpr int kMaxExperts = 1024;   // as the reference (moe_gate.cu:33)
constexpr int kMaxTopK = 32;        // as the reference (moe_gate.cu:35)
constexpr int kInverseScratch = 4;  // the stream scratch that holds the map

inline ks_status_t check_pairs(const char* where, int64_t tokens, int top_k, int64_t* pairs) {
  if (tokens > 0 && top_k > 0 && tokens > INT32_MAX / top_k)
    KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, std::string(where) + ": num_tokens*top_k exceeds int32 limit");
  *pairs = tokens * static_cast<int64_t>(top_k);
  return KS_SUCCESS;
}

// inverse[ids[r]] = r for the rows whose id is in range; other entries are left.
void enqueue_inverse_permutation(int32_t* inverse, const int32_t* ids, int64_t pairs, cudaStream_t stream);

// Stable counting sort of `pairs` ids into `groups` groups (ks_moe_compute_permutation); with `rest`, ids outside
// [0, groups - 1) belong to the last group instead of being dropped.
ks_status_t enqueue_group_sort(const char* where, int32_t* sorted_ids, int32_t* offsets, const int32_t* ids, int64_t pairs,
                               int groups, bool rest, cudaStream_t stream);

// `row` if it is the row of pair `pair`, else -1.
__device__ __forceinline__ int32_t check_row(int32_t row, const int32_t* __restrict__ ids, int64_t pair, int64_t pairs) {
  return (row >= 0 && row < pairs && __ldg(ids + row) == pair) ? row : -1;
}

}  // namespace ksb
