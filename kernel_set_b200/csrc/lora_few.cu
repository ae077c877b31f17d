// Low-rank adapters for single tokens: y = y0 + s B (A x) for up to 8 rows of an adapter at a time.
//
// What counts here is latency: an adapter of rank 16 beside a 4096 x 4096 projection is 256 KB. One launch does both products. A
// cluster of CTAs has an item (up to 8 rows of one adapter): each takes a slice of K, leaves its partial sums [rank x 8] in
// every CTA's shared memory, and behind one cluster barrier each has the whole inner vectors, added in rank order, and
// computes a slice of the outputs. With few items several clusters share one: each does the first product again (A comes from
// L2) and gives a part of the outputs. B's slice is asked into L2 at the start.
//
// Products by mma.m16n8k16 with the factor as the 16-row operand and the rows as the 8 columns; its order of k inside a block of
// 32 is changed so that a lane's four pairs are 16 adjacent bytes, and its order of rows in the second product so that a
// lane ends up with 8 adjacent outputs of two rows. The inner vectors enter as a high and a low 16-bit part, scaled per row.
#include <algorithm>
#include <string>

#include "lora_tiles.cuh"
#include "sm100_host.cuh"
#include "sm100_lora.cuh"
#include "sm100_ptx.cuh"

namespace ksb {
namespace sm100 {
namespace {

constexpr int kFew = 8;                // rows of an item
constexpr int kFewWarps = 8;
constexpr int kFewThreads = kFewWarps * 32;
constexpr int kFewCluster = 8;
constexpr int kUnit = 64;              // outputs a warp takes at a time

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load16(const void* p, bool take) {
  return take ? __ldg(static_cast<const uint4*>(p)) : make_uint4(0u, 0u, 0u, 0u);
}

// RT: 16-rank tiles.
template <typename T, int RT>
__global__ void __launch_bounds__(kFewThreads, RT <= 2 ? 3 : (RT <= 4 ? 2 : 1)) lora_few_kernel(const __grid_constant__ LoraPass p, int S, int parts) {
  constexpr int kRanks = RT * 16;
  constexpr int kBlocks = (RT + 1) / 2;                       // 32-rank blocks of the second product
  constexpr int kH = kBlocks * 32 * kFew;
  constexpr int kSums = RT <= 4 ? kFewWarps : kFewWarps / 2;   // (two warps share one at rank 128: 48 KB hold no more)
  __shared__ __align__(16) float warp_sum[kSums][kRanks * kFew];
  __shared__ __align__(16) float part_sum[kFewCluster][kRanks * kFew];   // of the cluster's CTAs
  float* h = &warp_sum[0][0];   // the inner vectors, once the warps' sums have been added up
  static_assert(kH <= kSums * kRanks * kFew, "shared memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, s4 = lane & 3;
  const int rank = blockIdx.x % S;
  const int part = (blockIdx.x / S) % parts;
  const int64_t item = blockIdx.x / (S * parts);
  if (S > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // (waited for before the first remote store)
  grid_dependency_wait();
  const TilePlace f = find_tile<kFew>(p.offsets, p.adapters, p.rows, item);
  // outputs of this CTA, in units
  const int64_t units = (p.d_out + kUnit - 1) / kUnit;
  const int slot = part * S + rank;
  const int64_t unit0 = units * slot / (S * parts), unit1 = units * (slot + 1) / (S * parts);
  const bool work = f.adapter >= 0 && f.adapter < p.adapters;
  if (!work) {
    if (f.adapter == p.adapters && p.out != p.base)
      for (int r = 0; r < f.count; ++r) {
        const int64_t row = lora_row(p.ids, f.place + r, p.rows);
        if (row < 0) continue;
        const int64_t end = unit1 * kUnit < p.d_out ? unit1 * kUnit : p.d_out;
        for (int64_t c = unit0 * kUnit + threadIdx.x * 8; c < end; c += kFewThreads * 8)
          *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + row * p.ld_out + c) =
              *reinterpret_cast<const uint4*>(static_cast<const T*>(p.base) + row * p.ld_base + c);
      }
    if (S > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    return;   // (the whole cluster)
  }
  const T* a = static_cast<const T*>(p.u) + static_cast<int64_t>(f.adapter) * p.rank * p.d_in;
  const T* b = static_cast<const T*>(p.v) + static_cast<int64_t>(f.adapter) * p.rank * p.d_out;
  {
    const char* from = reinterpret_cast<const char*>(b + unit0 * kUnit * p.rank);
    const int64_t bytes = ((unit1 * kUnit < p.d_out ? unit1 * kUnit : p.d_out) - unit0 * kUnit) * p.rank * 2;
    for (int64_t at = threadIdx.x * 128; at < bytes; at += kFewThreads * 128)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(from + at));
  }
  const float scale = __ldg(p.scales + f.adapter);
  const int64_t my_row = g < f.count ? lora_row(p.ids, f.place + g, p.rows) : -1;   // row g of the item
  const T* x = static_cast<const T*>(p.in) + (my_row >= 0 ? my_row : 0) * p.ld_in;

  // ---- first product: blocks of 32 k, warp by warp ----
  const int64_t blocks = (p.d_in + 31) / 32;
  const int64_t block0 = blocks * rank / S, block1 = blocks * (rank + 1) / S;
  float acc[RT][4];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;
  constexpr int kAhead = RT <= 2 ? 2 : 1;
  for (int64_t blk = block0 + warp; blk < block1; blk += kAhead * kFewWarps) {
    uint4 xv[kAhead], av[kAhead][RT][2];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t k = (blk + u * kFewWarps) * 32 + s4 * 8;
      const bool in = blk + u * kFewWarps < block1 && k < p.d_in;
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int j = t * 16 + i * 8 + g;
          const bool take = in && j < p.rank;
          av[u][t][i] = load16(a + (take ? j * p.d_in + k : 0), take);
        }
      xv[u] = load16(x + (in ? k : 0), in && my_row >= 0);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const uint4 lo = av[u][t][0], hi = av[u][t][1];
        mma16816<T>(acc[t], lo.x, hi.x, lo.y, hi.y, xv[u].x, xv[u].y);
        mma16816<T>(acc[t], lo.z, hi.z, lo.w, hi.w, xv[u].z, xv[u].w);
      }
  }
  if (kSums < kFewWarps) {
    if (warp >= kSums)
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<float2*>(&warp_sum[warp - kSums][(t * 16 + g + 8 * i) * kFew + 2 * s4]) = make_float2(acc[t][2 * i], acc[t][2 * i + 1]);
    __syncthreads();
  }
  if (warp < kSums)
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float2* at = reinterpret_cast<float2*>(&warp_sum[warp][(t * 16 + g + 8 * i) * kFew + 2 * s4]);
        const float2 other = kSums < kFewWarps ? *at : make_float2(0.f, 0.f);
        *at = make_float2(acc[t][2 * i] + other.x, acc[t][2 * i + 1] + other.y);
      }
  if (S > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // (the others have begun)
  __syncthreads();
  for (int e = threadIdx.x; e < kRanks * kFew; e += kFewThreads) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kSums; ++w) v += warp_sum[w][e];
    const uint32_t at = smem_u32(&part_sum[rank][e]);
    if (S > 1)
      for (int c = 0; c < S; ++c)
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_map_shared(at, c)), "f"(v) : "memory");
    else
      part_sum[0][e] = v;
  }
  if (S > 1) cluster_sync();
  else __syncthreads();
  for (int e = threadIdx.x; e < kH; e += kFewThreads) {
    float v = 0.f;
    if (e < kRanks * kFew)
      for (int c = 0; c < S; ++c) v += part_sum[c][e];
    h[e] = v;
    if (p.inner != nullptr && slot == 0 && e / kFew < p.rank && e % kFew < f.count) {
      const int64_t row = lora_row(p.ids, f.place + e % kFew, p.rows);
      if (row >= 0) p.inner[row * p.rank + e / kFew] = v;
    }
  }
  __syncthreads();

  // ---- second product ----
  uint32_t hi[kBlocks][4], lo[kBlocks][4];
  float down, up;
  {
    float v[kBlocks][8], most = 0.f;
#pragma unroll
    for (int r = 0; r < kBlocks; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[r][i] = h[(r * 32 + s4 * 8 + i) * kFew + g];
        most = fmaxf(most, fabsf(v[r][i]));
      }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    row_scale(most, &down, &up);
#pragma unroll
    for (int r = 0; r < kBlocks; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f0 = v[r][2 * i] * down, f1 = v[r][2 * i + 1] * down;
        hi[r][i] = Pair<T>::pack(f0, f1);
        const float2 w = Pair<T>::unpack(hi[r][i]);
        lo[r][i] = Pair<T>::pack(f0 - w.x, f1 - w.y);
      }
  }
  // this lane's outputs are of the rows 2 s4 and 2 s4 + 1
  float c[2];
  int64_t out_row[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    c[i] = scale * __shfl_sync(0xffffffffu, up, (2 * s4 + i) * 4);
    out_row[i] = __shfl_sync(0xffffffffu, my_row, (2 * s4 + i) * 4);
  }
  for (int64_t unit = unit0 + warp; unit < unit1; unit += kFewWarps) {
    const int64_t n = unit * kUnit + g * 8;   // rows n .. n + 7 of B
    const bool in = n < p.d_out;
    uint4 y0[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      y0[i] = out_row[i] >= 0 && in ? *reinterpret_cast<const uint4*>(static_cast<const T*>(p.base) + out_row[i] * p.ld_base + n)
                                    : make_uint4(0u, 0u, 0u, 0u);
    float d[4][4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) d[t][i] = 0.f;
#pragma unroll
    for (int r = 0; r < kBlocks; ++r) {
      uint4 w[8];
      const int j = r * 32 + s4 * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool take = in && j < p.rank;
        w[i] = load16(b + (take ? (n + i) * p.rank + j : 0), take);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint4 e = w[2 * t], o = w[2 * t + 1];
        mma16816<T>(d[t], e.x, o.x, e.y, o.y, hi[r][0], hi[r][1]);
        mma16816<T>(d[t], e.z, o.z, e.w, o.w, hi[r][2], hi[r][3]);
        mma16816<T>(d[t], e.x, o.x, e.y, o.y, lo[r][0], lo[r][1]);
        mma16816<T>(d[t], e.z, o.z, e.w, o.w, lo[r][2], lo[r][3]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (out_row[i] < 0 || !in) continue;
      uint32_t y[4] = {y0[i].x, y0[i].y, y0[i].z, y0[i].w};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float2 v = Pair<T>::unpack(y[t]);
        y[t] = Pair<T>::pack(fmaf(c[i], d[t][i], v.x), fmaf(c[i], d[t][2 + i], v.y));
      }
      *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + out_row[i] * p.ld_out + n) = make_uint4(y[0], y[1], y[2], y[3]);
    }
  }
}

}  // namespace

ks_status_t lora_few_pass(const char* where, const LoraPass& p, ks_dtype_t dtype, cudaStream_t stream) {
  const int64_t items = lora_tile_bound(p.rows, p.adapters, kFew);
  const int64_t room = static_cast<int64_t>(sm_count()) * 2;
  int s = kFewCluster;
  while (s > 1 && (p.d_in < 64 * s || items * s > 8 * room)) s /= 2;
  // several clusters per item while SMs are idle and the second product is still the larger part of each
  int parts = 1;
  while (items * s * parts * 2 <= room && p.d_out >= 2 * parts * p.d_in && p.d_out >= int64_t(kUnit) * s * parts * 2) parts *= 2;
  if (items * s * parts > INT32_MAX) KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, std::string(where) + ": grid exceeds CUDA grid limits");
  const unsigned grid = static_cast<unsigned>(items * s * parts);
#define KSB_LORA_FEW(T, RT) launch_programmatic_cluster(lora_few_kernel<T, RT>, grid, s, true, kFewThreads, 0, stream, p, s, parts)
#define KSB_LORA_FEW_T(T)                     \
  do {                                        \
    if (p.rank <= 16) KSB_LORA_FEW(T, 1);     \
    else if (p.rank <= 32) KSB_LORA_FEW(T, 2); \
    else if (p.rank <= 64) KSB_LORA_FEW(T, 4); \
    else KSB_LORA_FEW(T, 8);                  \
  } while (0)
  if (dtype == KS_DTYPE_F16) KSB_LORA_FEW_T(__half);
  else KSB_LORA_FEW_T(__nv_bfloat16);
#undef KSB_LORA_FEW_T
#undef KSB_LORA_FEW
  KSB_CHECK_LAUNCH(where);
  return KS_SUCCESS;
}

}  // namespace sm100
}  // namespace ksb
