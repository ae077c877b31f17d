// Low-rank adapters of many requests beside a shared projection, and their gradient: the entry points, and kernels
// for any shape. The reference has no operator of this kind; the formulas are in kernel_set/ext/lora.h.
//
// The forward pass and the gradient of the input are the same pair of products with the factors' roles changed
// (LoraPass): y = y0 + s V (U x), the inner vector U x of `rank` numbers held in fp32.
#include <string>

#include "common.cuh"
#include "kernel_set/ext/lora.h"
#include "lora_math.cuh"
#include "moe_rows.cuh"
#include "sm100_host.cuh"
#include "sm100_lora.cuh"
#include "sm100_ptx.cuh"

namespace ksb {
namespace {

constexpr int kMaxAnyRank = 4096;
constexpr int kAnyThreads = 256;
// Rows up to which the forward pass takes 8 to 32 at a time instead of tiles of 128, by rank (us cold, few / tiles): rank 16, 512 rows of 64
// adapters beside 4096 x 14336 43 / 68, of one beside 4096 x 4096 18.5 / 22.5; rank 32, 700 rows of 64 33 / 35, 1024 rows 37 / 35;
// rank 64, 256 rows of 64 35 / 39, 300 of 8 31 / 23, 512 of 64 43 / 39; rank 128, 200 of 8 35 / 27. Rows an adapter and widths move the
// border, which the rule does not see: rank 16, 1000 rows of 300 adapters 74 / 92, of 4 of 64 27 / 31, of 64 beside 1024 x 1024 27 / 16.
constexpr int few_rows(int rank) { return rank <= 32 ? 512 : 256; }

// Any rank, widths and alignment: a CTA per place. The warps take the ranks in turn, a lane every 32nd product of a
// sum; then a thread takes every 256th output.
template <typename T>
__global__ void __launch_bounds__(kAnyThreads) lora_any_kernel(LoraPass p) {
  extern __shared__ float inner[];   // [rank]
  sm100::grid_dependency_wait();
  const int64_t place = blockIdx.x;
  const int64_t row = lora_row(p.ids, place, p.rows);
  if (row < 0) return;
  const int a = lora_adapter(p.offsets, p.adapters, place, p.rows);
  if (a < 0) return;
  const T* base = static_cast<const T*>(p.base) + row * p.ld_base;
  T* out = static_cast<T*>(p.out) + row * p.ld_out;
  if (a >= p.adapters) {
    if (p.out != p.base)
      for (int64_t o = threadIdx.x; o < p.d_out; o += kAnyThreads) out[o] = base[o];
    return;
  }
  const T* in = static_cast<const T*>(p.in) + row * p.ld_in;
  const T* u = static_cast<const T*>(p.u) + static_cast<int64_t>(a) * p.rank * p.d_in;
  const T* v = static_cast<const T*>(p.v) + static_cast<int64_t>(a) * p.rank * p.d_out;
  const float s = __ldg(p.scales + a);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int j = warp; j < p.rank; j += kAnyThreads / 32) {
    float sum = 0.f;
    for (int64_t i = lane; i < p.d_in; i += 32) sum = fmaf(to_f32<T>(u[j * p.u_j + i * p.u_i]), to_f32<T>(in[i]), sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      inner[j] = sum;
      if (p.inner != nullptr) p.inner[row * p.rank + j] = p.scale_inner ? s * sum : sum;
    }
  }
  __syncthreads();
  for (int64_t o = threadIdx.x; o < p.d_out; o += kAnyThreads) {
    float sum = 0.f;
    for (int j = 0; j < p.rank; ++j) sum = fmaf(to_f32<T>(v[o * p.v_o + j * p.v_j]), inner[j], sum);
    out[o] = from_f32<T>(fmaf(s, sum, to_f32<T>(base[o])));
  }
}

// The factors' gradients for any shape: a thread per element, the adapter's rows in order.
template <typename T>
__global__ void __launch_bounds__(kAnyThreads) lora_weight_grad_any_kernel(LoraWeightGrad p) {
  sm100::grid_dependency_wait();
  const int a = blockIdx.y;
  const int64_t begin = lora_offset(p.offsets, a, p.rows), end = lora_offset(p.offsets, a + 1, p.rows);
  const float s = __ldg(p.scales + a);
  const int64_t in_a = p.k * p.rank, in_b = p.n * p.rank;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * kAnyThreads + threadIdx.x; e < in_a + in_b;
       e += static_cast<int64_t>(gridDim.x) * kAnyThreads) {
    const bool first = e < in_a;
    const int64_t at = first ? e : e - in_a;
    const int64_t j = first ? at / p.k : at % p.rank, i = first ? at % p.k : at / p.rank;
    const T* m = static_cast<const T*>(first ? p.x : p.d_out) + i;
    const int64_t ld = first ? p.ld_x : p.ld_d_out;
    const float* f = (first ? p.g : p.h) + j;
    float sum = 0.f;
    for (int64_t place = begin; place < end; ++place) {
      const int64_t row = lora_row(p.ids, place, p.rows);
      if (row >= 0) sum = fmaf(to_f32<T>(m[row * ld]), f[row * p.rank], sum);
    }
    if (first) static_cast<T*>(p.d_a)[a * in_a + at] = from_f32<T>(sum);
    else static_cast<T*>(p.d_b)[a * in_b + at] = from_f32<T>(s * sum);
  }
}

ks_status_t run_pass(const char* where, const LoraPass& p, bool forward, ks_dtype_t dtype, cudaStream_t s) {
  if (sm100::lora_tile_takes(p)) {
    if (forward && p.rows <= few_rows(p.rank)) return sm100::lora_few_pass(where, p, dtype, s);
    return sm100::lora_tile_pass(where, p, forward, dtype, s);
  }
  const unsigned grid = static_cast<unsigned>(p.rows);
  const size_t smem = static_cast<size_t>(p.rank) * sizeof(float);
  if (dtype == KS_DTYPE_F16) sm100::launch_programmatic(lora_any_kernel<__half>, grid, kAnyThreads, smem, s, p);
  else sm100::launch_programmatic(lora_any_kernel<__nv_bfloat16>, grid, kAnyThreads, smem, s, p);
  KSB_CHECK_LAUNCH(where);
  return KS_SUCCESS;
}

ks_status_t run_weight_grad(const char* where, const LoraWeightGrad& p, ks_dtype_t dtype, cudaStream_t s) {
  const int64_t blocks = ((p.k + p.n) * p.rank + kAnyThreads - 1) / kAnyThreads;
  const dim3 grid(static_cast<unsigned>(blocks < 65536 ? blocks : 65536), static_cast<unsigned>(p.adapters));
  if (dtype == KS_DTYPE_F16) sm100::launch_programmatic(lora_weight_grad_any_kernel<__half>, grid, kAnyThreads, 0, s, p);
  else sm100::launch_programmatic(lora_weight_grad_any_kernel<__nv_bfloat16>, grid, kAnyThreads, 0, s, p);
  KSB_CHECK_LAUNCH(where);
  return KS_SUCCESS;
}

// What both directions ask of their sizes.
ks_status_t check_sizes(const char* where, int64_t rows, int adapters, int rank, int64_t k, int64_t n, ks_dtype_t dtype) {
  const std::string w(where);
  if (rows < 0 || adapters <= 0 || rank <= 0 || k <= 0 || n <= 0) KSB_FAIL(KS_ERROR_INVALID_ARGUMENT, w + ": bad shape");
  if (rows > INT32_MAX) KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, w + ": num_tokens exceeds int32 limit");
  if (adapters > kMaxExperts - 1) KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, w + ": at most 1023 adapters");
  if (rank > kMaxAnyRank) KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, w + ": rank at most 4096");
  if (k > INT32_MAX / 2 || n > INT32_MAX / 2) KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, w + ": width exceeds int32 limit");
  if (dtype != KS_DTYPE_F16 && dtype != KS_DTYPE_BF16) KSB_FAIL(KS_ERROR_UNSUPPORTED_DTYPE, w + ": f16 or bf16 only");
  return KS_SUCCESS;
}

// The workspace of the backward pass: g [rows, rank], then two ranges per row for f16 (LoraPass).
int64_t inner_bytes(int64_t rows, int rank) { return (rows * rank * static_cast<int64_t>(sizeof(float)) + 255) / 256 * 256; }
int64_t workspace_bytes_of(int64_t rows, int rank) {
  return inner_bytes(rows, rank) + (2 * rows * static_cast<int64_t>(sizeof(float2)) + 255) / 256 * 256;
}

}  // namespace
}  // namespace ksb

using namespace ksb;

extern "C" {

ks_status_t ks_lora_plan(int32_t* sorted_ids, int32_t* offsets, const int32_t* adapter_ids, int64_t num_tokens,
                         int num_adapters, ks_stream_t stream) {
  const char* where = "ks_lora_plan";
  KSB_REQUIRE_PTR(offsets);
  if (num_tokens != 0) {   // (an empty tensor has no address)
    KSB_REQUIRE_PTR(sorted_ids);
    KSB_REQUIRE_PTR(adapter_ids);
  }
  if (num_tokens < 0 || num_adapters <= 0) KSB_FAIL(KS_ERROR_INVALID_ARGUMENT, "ks_lora_plan: bad shape");
  if (num_adapters > kMaxExperts - 1) KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, "ks_lora_plan: at most 1023 adapters");
  if (num_tokens > INT32_MAX) KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, "ks_lora_plan: num_tokens exceeds int32 limit");
  const ks_status_t st = require_sm100(where);
  if (st != KS_SUCCESS) return st;
  return enqueue_group_sort(where, sorted_ids, offsets, adapter_ids, num_tokens, num_adapters + 1, true, as_stream(stream));
}

ks_status_t ks_lora_apply(void* out, int64_t ld_out, const void* base, int64_t ld_base, float* h, const void* x, int64_t ld_x,
                          const void* a, const void* b, const float* scales, const int32_t* sorted_ids,
                          const int32_t* offsets, int64_t num_tokens, int num_adapters, int rank, int64_t k, int64_t n,
                          ks_dtype_t dtype, ks_stream_t stream) {
  const char* where = "ks_lora_apply";
  KSB_REQUIRE_PTR(a);
  KSB_REQUIRE_PTR(b);
  KSB_REQUIRE_PTR(scales);
  KSB_REQUIRE_PTR(offsets);
  if (num_tokens != 0) {   // (an empty tensor has no address)
    KSB_REQUIRE_PTR(out);
    KSB_REQUIRE_PTR(base);
    KSB_REQUIRE_PTR(x);
  }
  ks_status_t st = check_sizes(where, num_tokens, num_adapters, rank, k, n, dtype);
  if (st != KS_SUCCESS) return st;
  if (ld_x < k || ld_base < n || ld_out < n)
    KSB_FAIL(KS_ERROR_INVALID_ARGUMENT, "ks_lora_apply: a row is longer than its leading dimension");
  if (num_tokens == 0) return KS_SUCCESS;
  if (out == base && ld_out != ld_base)
    KSB_FAIL(KS_ERROR_INVALID_ARGUMENT, "ks_lora_apply: in place, ld_out and ld_base must be equal");
  if (out == x) KSB_FAIL(KS_ERROR_INVALID_ARGUMENT, "ks_lora_apply: out must not be x");
  st = require_sm100(where);
  if (st != KS_SUCCESS) return st;
  st = poll_kernel_fault(where);
  if (st != KS_SUCCESS) return st;
  LoraPass p = {};
  p.out = out; p.base = base; p.in = x; p.u = a; p.v = b; p.scales = scales; p.ids = sorted_ids; p.offsets = offsets;
  p.inner = h;
  p.ld_out = ld_out; p.ld_base = ld_base; p.ld_in = ld_x;
  p.rows = num_tokens; p.d_in = k; p.d_out = n;
  p.u_j = k; p.u_i = 1; p.v_o = rank; p.v_j = 1;
  p.adapters = num_adapters; p.rank = rank; p.scale_inner = false;
  return run_pass(where, p, true, dtype, as_stream(stream));
}

ks_status_t ks_lora_backward_workspace(size_t* bytes, int64_t num_tokens, int num_adapters, int rank, int64_t k, int64_t n) {
  KSB_REQUIRE_PTR(bytes);
  const ks_status_t st = check_sizes("ks_lora_backward_workspace", num_tokens, num_adapters, rank, k, n, KS_DTYPE_F16);
  if (st != KS_SUCCESS) return st;
  *bytes = static_cast<size_t>(workspace_bytes_of(num_tokens, rank));
  return KS_SUCCESS;
}

ks_status_t ks_lora_backward(void* d_x, int64_t ld_d_x, void* d_a, void* d_b, const void* d_x_base, int64_t ld_d_x_base,
                             const void* d_out, int64_t ld_d_out, const void* x, int64_t ld_x, const float* h, const void* a,
                             const void* b, const float* scales, const int32_t* sorted_ids, const int32_t* offsets,
                             int64_t num_tokens, int num_adapters, int rank, int64_t k, int64_t n, void* workspace,
                             size_t workspace_bytes, ks_dtype_t dtype, ks_stream_t stream) {
  const char* where = "ks_lora_backward";
  if (num_tokens != 0) {   // (an empty tensor has no address)
    KSB_REQUIRE_PTR(d_x);
    KSB_REQUIRE_PTR(d_x_base);
    KSB_REQUIRE_PTR(d_out);
    KSB_REQUIRE_PTR(x);
    KSB_REQUIRE_PTR(h);
  }
  KSB_REQUIRE_PTR(d_a);
  KSB_REQUIRE_PTR(d_b);
  KSB_REQUIRE_PTR(a);
  KSB_REQUIRE_PTR(b);
  KSB_REQUIRE_PTR(scales);
  KSB_REQUIRE_PTR(offsets);
  ks_status_t st = check_sizes(where, num_tokens, num_adapters, rank, k, n, dtype);
  if (st != KS_SUCCESS) return st;
  if (ld_x < k || ld_d_x < k || ld_d_x_base < k || ld_d_out < n)
    KSB_FAIL(KS_ERROR_INVALID_ARGUMENT, "ks_lora_backward: a row is longer than its leading dimension");
  if (num_tokens > 0 && d_x == d_x_base && ld_d_x != ld_d_x_base)
    KSB_FAIL(KS_ERROR_INVALID_ARGUMENT, "ks_lora_backward: in place, ld_d_x and ld_d_x_base must be equal");
  if (num_tokens > 0 && (d_x == d_out || d_x == x))
    KSB_FAIL(KS_ERROR_INVALID_ARGUMENT, "ks_lora_backward: d_x must be neither d_out nor x");
  const size_t want = static_cast<size_t>(workspace_bytes_of(num_tokens, rank));
  if (want > 0 && (workspace == nullptr || workspace_bytes < want || !aligned16(workspace)))
    KSB_FAIL(KS_ERROR_INVALID_ARGUMENT, "ks_lora_backward: workspace missing, too small or not 16-byte aligned");
  st = require_sm100(where);
  if (st != KS_SUCCESS) return st;
  st = poll_kernel_fault(where);
  if (st != KS_SUCCESS) return st;
  cudaStream_t s = as_stream(stream);
  float* g = static_cast<float*>(workspace);
  LoraPass p = {};
  p.out = d_x; p.base = d_x_base; p.in = d_out; p.u = b; p.v = a; p.scales = scales; p.ids = sorted_ids; p.offsets = offsets;
  p.inner = g;
  p.ld_out = ld_d_x; p.ld_base = ld_d_x_base; p.ld_in = ld_d_out;
  p.rows = num_tokens; p.d_in = n; p.d_out = k;
  p.u_j = 1; p.u_i = rank; p.v_o = 1; p.v_j = k;
  p.adapters = num_adapters; p.rank = rank; p.scale_inner = true;
  LoraWeightGrad w = {};
  w.d_a = d_a; w.d_b = d_b; w.x = x; w.d_out = d_out; w.g = g; w.h = h; w.scales = scales; w.ids = sorted_ids; w.offsets = offsets;
  w.ld_x = ld_x; w.ld_d_out = ld_d_out; w.rows = num_tokens; w.k = k; w.n = n; w.adapters = num_adapters; w.rank = rank;
  const bool tensor = sm100::lora_tile_takes(p) && sm100::lora_weight_grad_takes(w);
  if (tensor && dtype == KS_DTYPE_F16 && num_tokens > 0) {
    p.h = h;
    w.range_g = p.range_g = reinterpret_cast<float2*>(static_cast<char*>(workspace) + inner_bytes(num_tokens, rank));
    w.range_h = p.range_h = p.range_g + num_tokens;
  }
  if (num_tokens > 0) {
    st = run_pass(where, p, false, dtype, s);
    if (st != KS_SUCCESS) return st;
  }
  return tensor ? sm100::lora_weight_grad_pass(where, w, dtype, s) : run_weight_grad(where, w, dtype, s);
}

}  // extern "C"
