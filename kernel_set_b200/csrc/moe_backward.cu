// Gradients of a routed layer's steps: the gate's (softmax, top-k, weights optionally renormalised), the row
// gather's and the weighted sum's. No counterpart in the reference's C ABI.
//
// All three are bound by memory: a row is read and written once, sums are held in fp32 and rounded once, and every
// sum has one order (slots in turn; threads of a CTA by a fixed tree), so results repeat to the bit.
#include <string>
#include <type_traits>

#include "common.cuh"
#include "kernel_set/ext/moe_backward.h"
#include "moe_rows.cuh"
#include "sm100_host.cuh"
#include "sm100_ptx.cuh"

namespace ksb {
namespace {

// VEC consecutive elements, loaded and stored as one access where that is 16 bytes.
template <typename T, int VEC>
struct Piece {
  T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ Piece<T, VEC> load_piece(const T* p) {
  Piece<T, VEC> r;
  if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(r.v) = *reinterpret_cast<const uint4*>(p);
  else
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.v[i] = p[i];
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_piece(T* p, const Piece<T, VEC>& r) {
  if constexpr (VEC * sizeof(T) == 16) __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(r.v));
  else
#pragma unroll
    for (int i = 0; i < VEC; ++i) p[i] = r.v[i];
}

// ---------------------------------------------------------------------------------
// unpermute: out_t = sum_k w_tk p_r(t,k)  ->  dp_r = w_tk dout_t, dw_tk = <dout_t, p_r>
// ---------------------------------------------------------------------------------
// A CTA per sorted row. A pair without a row has no CTA that would write its weight's gradient; the first `zero_ctas`
// CTAs look for such pairs, kZeroPairs each: a bit per pair, set for every id among the rows, and a zero for each pair
// whose bit stayed clear. (A launch of its own to clear d_weights costs a small call a third of its time.)
constexpr int kRowThreads = 128;
constexpr int kZeroPairs = 32768;

__device__ __forceinline__ void zero_absent_pairs(float* __restrict__ d_weights, const int32_t* __restrict__ ids,
                                                  int64_t pairs, int64_t first, uint32_t* present) {
  for (int i = threadIdx.x; i < kZeroPairs / 32; i += kRowThreads) present[i] = 0u;
  __syncthreads();
  for (int64_t base = threadIdx.x; base < pairs; base += 8 * kRowThreads) {
    int32_t id[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t i = base + static_cast<int64_t>(j) * kRowThreads;
      id[j] = i < pairs ? __ldg(ids + i) : -1;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t at = static_cast<int64_t>(id[j]) - first;
      if (at >= 0 && at < kZeroPairs) atomicOr(present + (at >> 5), 1u << (at & 31));
    }
  }
  __syncthreads();
  const int64_t last = first + kZeroPairs < pairs ? first + kZeroPairs : pairs;
  for (int64_t i = first + threadIdx.x; i < last; i += kRowThreads)
    if (!(present[(i - first) >> 5] >> ((i - first) & 31) & 1u)) d_weights[i] = 0.f;
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kRowThreads)
unpermute_backward_kernel(T* d_permuted, float* __restrict__ d_weights, const T* __restrict__ d_out, const T* permuted,
                          const int32_t* __restrict__ ids, const float* __restrict__ weights, int64_t pairs, int top_k,
                          int64_t hidden, unsigned zero_ctas) {
  __shared__ uint32_t present[kZeroPairs / 32];
  __shared__ float parts[kRowThreads / 32];
  sm100::grid_dependency_wait();
  if (blockIdx.x < zero_ctas) {
    zero_absent_pairs(d_weights, ids, pairs, static_cast<int64_t>(blockIdx.x) * kZeroPairs, present);
    return;
  }
  const int64_t r = blockIdx.x - zero_ctas;
  const int32_t pair = __ldg(ids + r);
  const int64_t pieces = hidden / VEC;
  T* dp = d_permuted + r * hidden;
  if (pair < 0 || pair >= pairs) {
    Piece<T, VEC> zero;
#pragma unroll
    for (int i = 0; i < VEC; ++i) zero.v[i] = from_f32<T>(0.f);
    for (int64_t c = threadIdx.x; c < pieces; c += kRowThreads) store_piece<T, VEC>(dp + c * VEC, zero);
    return;
  }
  const float w = __ldg(weights + pair);
  const T* g = d_out + static_cast<int64_t>(pair / top_k) * hidden;
  const T* p = permuted + r * hidden;
  float dot = 0.f;
  constexpr int kAhead = 4;   // pieces of both rows in flight
  for (int64_t c0 = threadIdx.x; c0 < pieces; c0 += kAhead * kRowThreads) {
    Piece<T, VEC> gv[kAhead], pv[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t c = c0 + u * kRowThreads;
      if (c < pieces) {
        pv[u] = load_piece<T, VEC>(p + c * VEC);
        gv[u] = load_piece<T, VEC>(g + c * VEC);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t c = c0 + u * kRowThreads;
      if (c >= pieces) continue;
      Piece<T, VEC> o;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = to_f32<T>(gv[u].v[i]);
        dot = fmaf(d, to_f32<T>(pv[u].v[i]), dot);
        o.v[i] = from_f32<T>(w * d);
      }
      store_piece<T, VEC>(dp + c * VEC, o);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
  if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = dot;
  __syncthreads();
  if (threadIdx.x == 0) {
    float sum = parts[0];
#pragma unroll
    for (int i = 1; i < kRowThreads / 32; ++i) sum += parts[i];
    d_weights[pair] = sum;
  }
}

// ---------------------------------------------------------------------------------
// permute: p_r = x_t  ->  dx_t = sum over the rows r of t of dp_r
// ---------------------------------------------------------------------------------
// A CTA takes kRowThreads pieces of a token; its rows' numbers go through shared memory once, then eight slots'
// pieces are in flight together. Where the rows lie: up to kScanPairs pairs a CTA looks through all ids itself (16 KB from
// L2, no second launch); beyond that they come from the inverse map, looked up again as ks_moe_unpermute does.
constexpr int kScanPairs = 4096;

template <typename T, int VEC, bool SCAN>
__global__ void __launch_bounds__(kRowThreads)
permute_backward_kernel(T* __restrict__ d_input, const T* __restrict__ d_permuted, const int32_t* __restrict__ ids,
                        const int32_t* __restrict__ inverse, int64_t pairs, int top_k, int64_t hidden, unsigned chunks) {
  extern __shared__ int32_t rows[];   // of the token's slots
  sm100::grid_dependency_wait();
  const int64_t token = blockIdx.x / chunks;
  const int64_t c = static_cast<int64_t>(blockIdx.x - token * chunks) * kRowThreads + threadIdx.x;
  const int64_t first = token * top_k;
  if (SCAN) {
    for (int k = threadIdx.x; k < top_k; k += kRowThreads) rows[k] = -1;
    __syncthreads();
    for (int64_t base = threadIdx.x; base < pairs; base += 8 * kRowThreads) {
      int32_t id[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t i = base + j * kRowThreads;
        id[j] = i < pairs ? __ldg(ids + i) : -1;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (id[j] >= first && id[j] < first + top_k) rows[id[j] - first] = static_cast<int32_t>(base + j * kRowThreads);
    }
  } else {
    for (int k = threadIdx.x; k < top_k; k += kRowThreads)
      rows[k] = check_row(__ldg(inverse + first + k), ids, first + k, pairs);
  }
  __syncthreads();
  if (c >= hidden / VEC) return;
  float acc[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
  for (int k0 = 0; k0 < top_k; k0 += 8) {
    Piece<T, VEC> v[8];
    int32_t row[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      row[j] = k0 + j < top_k ? rows[k0 + j] : -1;
      if (row[j] >= 0) v[j] = load_piece<T, VEC>(d_permuted + static_cast<int64_t>(row[j]) * hidden + c * VEC);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (row[j] >= 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += to_f32<T>(v[j].v[i]);
      }
  }
  Piece<T, VEC> o;
#pragma unroll
  for (int i = 0; i < VEC; ++i) o.v[i] = from_f32<T>(acc[i]);
  store_piece<T, VEC>(d_input + token * hidden + c * VEC, o);
}

// ---------------------------------------------------------------------------------
// gate
// ---------------------------------------------------------------------------------
// A warp per token, lane l has the experts l, l + 32, ...; every lane adds the slots of its experts up in turn,
// from registers of the lanes that hold them.
template <typename T>
__global__ void __launch_bounds__(256)
gate_backward_kernel(T* d_logits, const float* __restrict__ d_weights, const float* __restrict__ weights,
                     const int32_t* __restrict__ indices, const T* logits, int64_t tokens, int experts, int top_k,
                     int renormalize) {
  sm100::grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (token >= tokens) return;   // whole warp
  int idx = -1;
  float w = 0.f, dw = 0.f;
  if (lane < top_k) {
    idx = __ldg(indices + token * top_k + lane);
    if (idx >= 0 && idx < experts) {
      w = __ldg(weights + token * top_k + lane);
      dw = __ldg(d_weights + token * top_k + lane);
    } else {
      idx = -1;
    }
  }
  float s = w * dw;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const float add = renormalize ? w * (dw - s) : w * dw;
  const T* row = logits + token * experts;
  float mx = -__int_as_float(0x7f800000), sum = 0.f;
  if (!renormalize) {
    for (int e = lane; e < experts; e += 32) mx = fmaxf(mx, to_f32<T>(row[e]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    for (int e = lane; e < experts; e += 32) sum += expf(to_f32<T>(row[e]) - mx);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  const float scale = renormalize ? 0.f : -s / sum;
  for (int e0 = 0; e0 < experts; e0 += 32) {
    const int e = e0 + lane;
    float d = renormalize || e >= experts ? 0.f : expf(to_f32<T>(row[e]) - mx) * scale;
    for (int k = 0; k < top_k; ++k) {
      const int ek = __shfl_sync(0xffffffffu, idx, k);
      const float ak = __shfl_sync(0xffffffffu, add, k);
      if (ek == e) d += ak;
    }
    if (e < experts) d_logits[token * experts + e] = from_f32<T>(d);
  }
}

}  // namespace
}  // namespace ksb

using namespace ksb;

namespace {

// Whether rows of `hidden` elements can be taken 16 bytes at a time.
bool rows16(int64_t hidden, int64_t elt, const void* a, const void* b, const void* c = nullptr) {
  return hidden * elt % 16 == 0 && aligned16(a) && aligned16(b) && aligned16(c);
}

template <typename T>
ks_status_t unpermute_backward(void* d_permuted, float* d_weights, const void* d_out, const void* permuted, const int32_t* ids,
                               const float* weights, int64_t pairs, int top_k, int64_t hidden, cudaStream_t s) {
  constexpr int kVec = 16 / sizeof(T);
  const unsigned zero_ctas = static_cast<unsigned>((pairs + kZeroPairs - 1) / kZeroPairs);
  const dim3 grid(static_cast<unsigned>(pairs) + zero_ctas);
  const auto kernel = rows16(hidden, sizeof(T), d_permuted, d_out, permuted) ? unpermute_backward_kernel<T, kVec>
                                                                            : unpermute_backward_kernel<T, 1>;
  sm100::launch_programmatic(kernel, grid, kRowThreads, 0, s, static_cast<T*>(d_permuted), d_weights,
                             static_cast<const T*>(d_out), static_cast<const T*>(permuted), ids, weights, pairs, top_k, hidden,
                             zero_ctas);
  KSB_CHECK_LAUNCH("ks_moe_unpermute_backward");
  return KS_SUCCESS;
}

template <typename T>
ks_status_t permute_backward(void* d_input, const void* d_permuted, const int32_t* ids, int64_t tokens, int top_k,
                             int64_t hidden, cudaStream_t s) {
  const char* where = "ks_moe_permute_backward";
  constexpr int kVec = 16 / sizeof(T);
  const int64_t pairs = tokens * top_k;
  const bool vec = rows16(hidden, sizeof(T), d_input, d_permuted);
  const int64_t pieces = vec ? hidden / kVec : hidden;
  const int64_t chunks = (pieces + kRowThreads - 1) / kRowThreads;
  if (chunks > INT32_MAX / tokens) KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, "ks_moe_permute_backward: grid exceeds CUDA grid limits");
  const unsigned grid = static_cast<unsigned>(tokens * chunks);
  const size_t smem = static_cast<size_t>(top_k) * sizeof(int32_t);
  T* o = static_cast<T*>(d_input);
  const T* x = static_cast<const T*>(d_permuted);
  if (pairs <= kScanPairs) {
    const auto kernel = vec ? permute_backward_kernel<T, kVec, true> : permute_backward_kernel<T, 1, true>;
    sm100::launch_programmatic(kernel, grid, kRowThreads, smem, s, o, x, ids, nullptr, pairs, top_k, hidden,
                               static_cast<unsigned>(chunks));
    KSB_CHECK_LAUNCH(where);
    return KS_SUCCESS;
  }
  sm100::StreamScratch scratch(s);   // (until both kernels are enqueued)
  int32_t* inverse = static_cast<int32_t*>(scratch.get(static_cast<size_t>(pairs) * sizeof(int32_t), kInverseScratch));
  if (inverse == nullptr) KSB_FAIL(KS_ERROR_OUT_OF_MEMORY, "ks_moe_permute_backward: workspace allocation failed");
  enqueue_inverse_permutation(inverse, ids, pairs, s);
  const auto kernel = vec ? permute_backward_kernel<T, kVec, false> : permute_backward_kernel<T, 1, false>;
  sm100::launch_programmatic(kernel, grid, kRowThreads, smem, s, o, x, ids, inverse, pairs, top_k, hidden,
                             static_cast<unsigned>(chunks));
  KSB_CHECK_LAUNCH(where);
  return KS_SUCCESS;
}

}  // namespace

extern "C" {

ks_status_t ks_moe_unpermute_backward(void* d_permuted, float* d_weights, const void* d_out, const void* permuted,
                                      const int32_t* sorted_token_ids, const float* routing_weights, int64_t num_tokens,
                                      int top_k, int64_t hidden, ks_dtype_t dtype, ks_stream_t stream) {
  const char* where = "ks_moe_unpermute_backward";
  if (num_tokens == 0 && top_k > 0 && hidden > 0) return KS_SUCCESS;   // (an empty tensor has no address)
  KSB_REQUIRE_PTR(d_permuted);
  KSB_REQUIRE_PTR(d_weights);
  KSB_REQUIRE_PTR(d_out);
  KSB_REQUIRE_PTR(permuted);
  KSB_REQUIRE_PTR(sorted_token_ids);
  KSB_REQUIRE_PTR(routing_weights);
  if (num_tokens < 0 || top_k <= 0 || hidden <= 0)
    KSB_FAIL(KS_ERROR_INVALID_ARGUMENT, "ks_moe_unpermute_backward: bad shape");
  if (d_permuted == d_out) KSB_FAIL(KS_ERROR_INVALID_ARGUMENT, "ks_moe_unpermute_backward: d_permuted must not be d_out");
  if (!is_float3(dtype)) KSB_FAIL(KS_ERROR_UNSUPPORTED_DTYPE, "ks_moe_unpermute_backward: unsupported dtype");
  int64_t pairs = 0;
  ks_status_t st = check_pairs(where, num_tokens, top_k, &pairs);
  if (st != KS_SUCCESS) return st;
  if (pairs + pairs / kZeroPairs + 1 > INT32_MAX)
    KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, "ks_moe_unpermute_backward: grid exceeds CUDA grid limits");
  st = require_sm100(where);
  if (st != KS_SUCCESS) return st;
  cudaStream_t s = as_stream(stream);
  const auto run = dtype == KS_DTYPE_F32 ? unpermute_backward<float>
                   : dtype == KS_DTYPE_F16 ? unpermute_backward<__half>
                                           : unpermute_backward<__nv_bfloat16>;
  return run(d_permuted, d_weights, d_out, permuted, sorted_token_ids, routing_weights, pairs, top_k, hidden, s);
}

ks_status_t ks_moe_permute_backward(void* d_input, const void* d_permuted, const int32_t* sorted_token_ids, int64_t num_tokens,
                                    int top_k, int64_t hidden, ks_dtype_t dtype, ks_stream_t stream) {
  const char* where = "ks_moe_permute_backward";
  if (num_tokens == 0 && top_k > 0 && hidden > 0) return KS_SUCCESS;   // (an empty tensor has no address)
  KSB_REQUIRE_PTR(d_input);
  KSB_REQUIRE_PTR(d_permuted);
  KSB_REQUIRE_PTR(sorted_token_ids);
  if (num_tokens < 0 || top_k <= 0 || hidden <= 0)
    KSB_FAIL(KS_ERROR_INVALID_ARGUMENT, "ks_moe_permute_backward: bad shape");
  if (top_k > 4096) KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, "ks_moe_permute_backward: top_k at most 4096");
  if (d_input == d_permuted) KSB_FAIL(KS_ERROR_INVALID_ARGUMENT, "ks_moe_permute_backward: d_input must not be d_permuted");
  if (!is_float3(dtype)) KSB_FAIL(KS_ERROR_UNSUPPORTED_DTYPE, "ks_moe_permute_backward: unsupported dtype");
  int64_t pairs = 0;
  ks_status_t st = check_pairs(where, num_tokens, top_k, &pairs);
  if (st != KS_SUCCESS) return st;
  st = require_sm100(where);
  if (st != KS_SUCCESS) return st;
  cudaStream_t s = as_stream(stream);
  const auto run = dtype == KS_DTYPE_F32 ? permute_backward<float>
                   : dtype == KS_DTYPE_F16 ? permute_backward<__half>
                                           : permute_backward<__nv_bfloat16>;
  return run(d_input, d_permuted, sorted_token_ids, num_tokens, top_k, hidden, s);
}

ks_status_t ks_moe_gate_softmax_topk_backward(void* d_logits, const float* d_weights, const float* weights,
                                              const int32_t* indices, const void* logits, int64_t num_tokens, int num_experts,
                                              int top_k, int renormalize, ks_dtype_t dtype, ks_stream_t stream) {
  const char* where = "ks_moe_gate_softmax_topk_backward";
  if (num_tokens == 0 && num_experts > 0 && top_k > 0 && top_k <= num_experts) return KS_SUCCESS;   // (an empty tensor has no address)
  KSB_REQUIRE_PTR(d_logits);
  KSB_REQUIRE_PTR(d_weights);
  KSB_REQUIRE_PTR(weights);
  KSB_REQUIRE_PTR(indices);
  if (!renormalize) KSB_REQUIRE_PTR(logits);
  if (num_tokens < 0 || num_experts <= 0 || top_k <= 0 || top_k > num_experts)
    KSB_FAIL(KS_ERROR_INVALID_ARGUMENT, "ks_moe_gate_softmax_topk_backward: bad shape");
  if (num_experts > kMaxExperts || top_k > kMaxTopK)
    KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, "ks_moe_gate_softmax_topk_backward: at most 1024 experts and top_k 32");
  if (!is_float3(dtype)) KSB_FAIL(KS_ERROR_UNSUPPORTED_DTYPE, "ks_moe_gate_softmax_topk_backward: unsupported dtype");
  if ((num_tokens + 7) / 8 > INT32_MAX)
    KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, "ks_moe_gate_softmax_topk_backward: grid exceeds CUDA grid limits");
  ks_status_t st = require_sm100(where);
  if (st != KS_SUCCESS) return st;
  cudaStream_t s = as_stream(stream);
  const dim3 grid(static_cast<unsigned>((num_tokens + 7) / 8));
#define KSB_GATE_BACKWARD(T)                                                                                        \
  sm100::launch_programmatic(gate_backward_kernel<T>, grid, 256, 0, s, static_cast<T*>(d_logits), d_weights, weights, \
                             indices, static_cast<const T*>(logits), num_tokens, num_experts, top_k, renormalize)
  if (dtype == KS_DTYPE_F32) KSB_GATE_BACKWARD(float);
  else if (dtype == KS_DTYPE_F16) KSB_GATE_BACKWARD(__half);
  else KSB_GATE_BACKWARD(__nv_bfloat16);
#undef KSB_GATE_BACKWARD
  KSB_CHECK_LAUNCH(where);
  return KS_SUCCESS;
}

}  // extern "C"
