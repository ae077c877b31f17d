// Layout of the adapters' problem, shared by the kernels for any shape and those for the tensor cores.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ksb {

// One product pair y = y0 + c V (U x) over rows sorted by adapter: the forward pass with U = A, V = B, the gradient of
// the input with U = B^T, V = A^T. U [L, rank, d_in] and V [L, d_out, rank] are given by the strides of their stored forms.
struct LoraPass {
  void* out;              // [rows, d_out]
  const void* base;       // the same
  const void* in;         // [rows, d_in]
  const void* u;          // adapter a, rank j, input i: u + a * rank * d_in + j * u_j + i * u_i
  const void* v;          // adapter a, output o, rank j: v + a * rank * d_out + o * v_o + j * v_j
  const float* scales;
  const int32_t* ids;     // may be NULL
  const int32_t* offsets;
  float* inner;           // [rows, rank] fp32, may be NULL: U x (forward), or s U x (backward)
  const float* h;         // with range_h: [rows, rank] fp32
  float2* range_g;        // may be NULL: [rows] by place; for every 32 places from the start of an adapter's on, at the first
  float2* range_h;        // of them, the largest and the smallest magnitude but zero of their rows in `inner` and in h
  int64_t ld_out, ld_base, ld_in;
  int64_t rows;
  int64_t d_in, d_out;
  int64_t u_j, u_i, v_o, v_j;
  int adapters, rank;
  bool scale_inner;       // whether `inner` holds s U x
};

// The gradients of the factors: for adapter a the sums over its rows
//   d_a[j, i] = sum g[row, j] x[row, i],   d_b[i, j] = scale sum dout[row, i] h[row, j].
struct LoraWeightGrad {
  void* d_a;
  void* d_b;
  const void* x;
  const void* d_out;
  const float* g;         // [rows, rank], scaled
  const float* h;         // [rows, rank]
  const float* scales;
  const int32_t* ids;
  const int32_t* offsets;
  const float2* range_g;  // as LoraPass's, for f16 on the tensor cores
  const float2* range_h;
  int64_t ld_x, ld_d_out;
  int64_t rows;
  int64_t k, n;
  int adapters, rank;
};

// Row at place p, -1 for none.
__device__ __forceinline__ int64_t lora_row(const int32_t* __restrict__ ids, int64_t p, int64_t rows) {
  if (ids == nullptr) return p;
  const int64_t r = __ldg(ids + p);
  return r >= 0 && r < rows ? r : -1;
}
// offsets[a] within [0, rows].
__device__ __forceinline__ int64_t lora_offset(const int32_t* __restrict__ offsets, int a, int64_t rows) {
  const int64_t o = __ldg(offsets + a);
  return o < 0 ? 0 : (o > rows ? rows : o);
}
// The adapter of place p: the last a with offsets[a] <= p, `adapters` when p lies behind the last one's rows, -1 in front of the first's.
__device__ __forceinline__ int lora_adapter(const int32_t* __restrict__ offsets, int adapters, int64_t p, int64_t rows) {
  int lo = -1, hi = adapters;   // offsets[lo] <= p (or lo = -1)
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (lora_offset(offsets, mid, rows) <= p) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

}  // namespace ksb
