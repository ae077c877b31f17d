/*
 * Low-rank adapters of many requests at once, beside a projection that they
 * share (a quantized GEMM of kernel_set/gemm.h, or the experts of a routed layer).
 *
 * Row t of the batch has adapter a(t), or none; adapter a has a scale s, A [rank, K]
 * and B [N, rank]:
 *   forward   h_t = A x_t,  out_t = base_t + s B h_t
 *   backward  g_t = s B^T d_out_t,  d_x_t = d_x_base_t + A^T g_t,
 *             d_A = sum_t g_t x_t^T,  d_B = s sum_t d_out_t h_t^T
 * Rows without an adapter keep their base. The rows are taken in the order of a
 * plan, sorted by adapter, that all layers of a step share.
 *
 * The reference has no operator of this kind. No entry point allocates or
 * synchronises.
 */
#ifndef KERNEL_SET_EXT_LORA_H_
#define KERNEL_SET_EXT_LORA_H_

#include "kernel_set/types.h"

KS_BEGIN_EXTERN_C

/*
 * Stable counting sort of the rows by adapter.
 *   adapter_ids  [num_tokens] int32; an id outside [0, num_adapters) is "none"
 *   sorted_ids   [num_tokens] int32: rows in adapter order, those without at the end
 *   offsets      [num_adapters + 2] int32: where each adapter's rows begin, where the
 *                rows without begin, num_tokens
 * At most 1023 adapters. One launch.
 */
KS_API ks_status_t ks_lora_plan(int32_t* sorted_ids, int32_t* offsets,
                                const int32_t* adapter_ids, int64_t num_tokens,
                                int num_adapters, ks_stream_t stream);

/*
 * out = base + s B (A x), row by row.
 *   x [num_tokens, k], base, out [num_tokens, n], a [num_adapters, rank, k],
 *   b [num_adapters, n, rank]: f16 or bf16 (`dtype`); scales [num_adapters] fp32
 *   ld_x, ld_base, ld_out: elements from a row to the next, at least k, n, n
 *   out may be base (then with the same ld); otherwise it overlaps nothing
 *   h            [num_tokens, rank] fp32 or NULL: receives A x for the rows that have an
 *                adapter (others keep what they held), which the backward pass reads
 *   sorted_ids   as ks_lora_plan gives them, or NULL: row i is at place i. Places with an
 *                id outside [0, num_tokens) are left out, and a row whose id is at no place
 *                is left as it was; a row may be at one place
 *   offsets      [num_adapters + 1], ascending: places offsets[a] .. offsets[a+1] have adapter a, places from
 *                offsets[num_adapters] on none; places in front of offsets[0] are left out (part of a longer
 *                table, as a rank's own experts'). Values are clamped to [0, num_tokens].
 * With ks_moe_compute_permutation's offsets and sorted_ids = NULL the rows of a routed
 * layer that are sorted by expert get their expert's adapter.
 * fp32 accumulation, one rounding to `dtype`; A x enters the second product in fp32 or as a sum of 16-bit
 * numbers that hold it to 2^-24 of each element (bf16), or to 2^-22 of each element and 2^-50 of the row's
 * largest, whichever is more (f16). A row whose A x is not finite gets NaN where
 * it would get infinities. rank at most 4096.
 */
KS_API ks_status_t ks_lora_apply(void* out, int64_t ld_out, const void* base,
                                 int64_t ld_base, float* h, const void* x,
                                 int64_t ld_x, const void* a, const void* b,
                                 const float* scales, const int32_t* sorted_ids,
                                 const int32_t* offsets, int64_t num_tokens,
                                 int num_adapters, int rank, int64_t k,
                                 int64_t n, ks_dtype_t dtype,
                                 ks_stream_t stream);

/* Bytes of the workspace that ks_lora_backward wants for these sizes. */
KS_API ks_status_t ks_lora_backward_workspace(size_t* bytes, int64_t num_tokens,
                                              int num_adapters, int rank,
                                              int64_t k, int64_t n);

/*
 * Gradient of ks_lora_apply.
 *   d_out [num_tokens, n], x, d_x_base, d_x [num_tokens, k], a, d_a [num_adapters, rank, k],
 *   b, d_b [num_adapters, n, rank]: `dtype`, f16 or bf16; h [num_tokens, rank] fp32 as the
 *   forward pass gave it; scales, sorted_ids, offsets, ld_* as there
 *   d_x may be d_x_base (the gradient through the shared projection is added to)
 *   d_a, d_b are written whole, with zeros for an adapter without rows
 *   workspace: 16-byte aligned device memory of the size above, undefined on entry and exit; two calls
 *   that may overlap need one each
 * d_out is the gradient of base as it is. Sums in fp32, one rounding. g and h enter the products as A x does in
 * ks_lora_apply; for d_a and d_b in f16 "largest" is the adapter's, and an adapter whose elements lie further apart than
 * 2^33 gets plain fp32 sums, as do, in both types, sums that are not finite (slow: 7.6 ms against 0.15 where that is all
 * of d_b for 16384 rows of rank 64 beside 4096 x 4096). A row whose g is not finite gets NaN in d_x where it would get
 * infinities. The same inputs and plan give the same bits; how the additions of d_a and d_b are grouped depends on the sizes
 * and on the adapter's number of rows.
 */
KS_API ks_status_t ks_lora_backward(
    void* d_x, int64_t ld_d_x, void* d_a, void* d_b, const void* d_x_base,
    int64_t ld_d_x_base, const void* d_out, int64_t ld_d_out, const void* x,
    int64_t ld_x, const float* h, const void* a, const void* b,
    const float* scales, const int32_t* sorted_ids, const int32_t* offsets,
    int64_t num_tokens, int num_adapters, int rank, int64_t k, int64_t n,
    void* workspace, size_t workspace_bytes, ks_dtype_t dtype,
    ks_stream_t stream);

KS_END_EXTERN_C

#endif /* KERNEL_SET_EXT_LORA_H_ */
