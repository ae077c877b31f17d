// The adapters' kernels for the tensor cores (sm100_lora.cu).
#pragma once

#include "common.cuh"
#include "lora_math.cuh"

namespace ksb {
namespace sm100 {

// Rows of a token tile.
constexpr int kLoraTile = 128;

// Tiles of `tile` rows that `rows` rows of `adapters` adapters can need: every adapter's last one may be partly filled, and so
// may that of the rows without one.
inline int64_t lora_tile_bound(int64_t rows, int adapters, int tile) {
  const int64_t groups = adapters + 1 < rows ? adapters + 1 : rows;
  return (rows - groups) / tile + groups;
}

// Whether the tile kernel takes the pass: 16-byte aligned rows, rank and widths multiples of 8, rank at most 128.
bool lora_tile_takes(const LoraPass& p);
// forward: U [rank, d_in], V [d_out, rank] as stored; otherwise U and V are the transposes of what is stored.
ks_status_t lora_tile_pass(const char* where, const LoraPass& p, bool forward, ks_dtype_t dtype, cudaStream_t stream);

// The forward pass of a few rows per adapter (single tokens): legacy tensor-core instructions with the rows as their 8 columns,
// under the same conditions.
ks_status_t lora_few_pass(const char* where, const LoraPass& p, ks_dtype_t dtype, cudaStream_t stream);

// The factors' gradients, where lora_tile_takes the pass before them and the gradients and x are 16-byte aligned.
bool lora_weight_grad_takes(const LoraWeightGrad& p);
ks_status_t lora_weight_grad_pass(const char* where, const LoraWeightGrad& p, ks_dtype_t dtype, cudaStream_t stream);

}  // namespace sm100
}  // namespace ksb
