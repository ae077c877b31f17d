// Low-rank adapters for single tokens and short prompts: y = y0 + s B (A x) for 8, 16 or 32 rows of an adapter at a time.
//
// What counts here is latency: an adapter of rank 16 beside a 4096 x 4096 projection is 256 KB. One launch does both products. A
// cluster of CTAs has an item (up to 32 rows of one adapter): each takes a slice of K, leaves its partial sums [rank x rows] in
// every CTA's shared memory, and behind one cluster barrier each has the whole inner vectors, added in rank order, and
// computes a slice of the outputs. With few items several clusters share one: each does the first product again (A comes from
// L2) and gives a part of the outputs. B's slice is asked into L2 at the start.
//
// Products by mma.m16n8k16 with the factor as the 16-row operand and 8 rows as the columns; its order of k inside a block of
// 32 is changed so that a lane's four pairs are 16 adjacent bytes, and its order of rows in the second product so that a
// lane ends up with 8 adjacent outputs of two rows. The inner vectors enter as 16-bit parts, scaled per row, the small parts first.
#include <mutex>
#include <string>
#include <type_traits>

#include "lora_tiles.cuh"
#include "sm100_host.cuh"
#include "sm100_lora.cuh"
#include "sm100_ptx.cuh"

namespace ksb {
namespace sm100 {
namespace {

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

// RT: 16-rank tiles, NT: groups of 8 rows of an item.
template <typename T, int RT, int NT>
struct FewCfg {
  static constexpr int kRows = 8 * NT;
  static constexpr int kRanks = RT * 16;
  static constexpr int kBlocks = (RT + 1) / 2;                          // 32-rank blocks of the second product
  static constexpr int kElems = kRanks * kRows;                         // of the inner vectors, [rank][row]
  static constexpr int kSums = RT * NT <= 8 ? kFewWarps : (RT * NT <= 16 ? 4 : 2);   // places for the warps' sums
  static constexpr int kParts = kSums * kElems * 4;                     // the cluster's sums lie behind them
  static constexpr int kFrag = kParts + kFewCluster * kElems * 4;       // 16-bit parts of the inner vectors, as operands
  static constexpr int kUp = kFrag + NT * kBlocks * kInnerParts<T> * 32 * 16;   // the rows' scales
  static constexpr int kSmem = kUp + kRows * 4;
  static constexpr int kPerSm = RT * NT == 1 ? 3 : (RT <= 4 ? 2 : 1);
  static_assert(kPerSm * (kSmem + 1024) <= 233472, "shared memory");
};

template <typename T, int RT, int NT>
__global__ void __launch_bounds__(kFewThreads, FewCfg<T, RT, NT>::kPerSm) lora_few_kernel(const __grid_constant__ LoraPass p, int s_log, int parts_log) {
  using C = FewCfg<T, RT, NT>;
  constexpr int kParts = kInnerParts<T>;
  extern __shared__ __align__(16) unsigned char few_smem[];
  float* warp_sum = reinterpret_cast<float*>(few_smem);
  float* part_sum = reinterpret_cast<float*>(few_smem + C::kParts);
  uint4* frag = reinterpret_cast<uint4*>(few_smem + C::kFrag);          // [group][block][part][lane]
  float* ups = reinterpret_cast<float*>(few_smem + C::kUp);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, s4 = lane & 3;
  const int S = 1 << s_log;                                             // CTAs of a cluster; 1 << parts_log clusters per item
  const int rank = blockIdx.x & (S - 1);
  const int slot = blockIdx.x & ((1 << (s_log + parts_log)) - 1);       // of the item's CTAs
  const int64_t item = blockIdx.x >> (s_log + parts_log);
  if (S > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // (waited for before the first remote store)
  grid_dependency_wait();
  const TilePlace f = find_tile<C::kRows>(p.offsets, p.adapters, p.rows, item);
  // outputs of this CTA, in units
  const int64_t units = (p.d_out + kUnit - 1) / kUnit;
  const int64_t unit0 = units * slot >> (s_log + parts_log), unit1 = units * (slot + 1) >> (s_log + parts_log);
  if (f.adapter < 0 || f.adapter >= p.adapters) {
    if (f.adapter == p.adapters && p.out != p.base) {
      const int64_t end = unit1 * kUnit < p.d_out ? unit1 * kUnit : p.d_out;
      for (int r = warp; r < f.count; r += kFewWarps) {
        const int64_t row = lora_row(p.ids, f.place + r, p.rows);
        if (row < 0) continue;
        for (int64_t c = unit0 * kUnit + lane * 8; c < end; c += 256)
          *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + row * p.ld_out + c) =
              *reinterpret_cast<const uint4*>(static_cast<const T*>(p.base) + row * p.ld_base + c);
      }
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
  const int groups = (f.count + 7) / 8;   // that hold rows
  int32_t my_row[NT];                     // row g of each group, -1 for none
  const T* x[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    my_row[n] = n * 8 + g < f.count ? static_cast<int32_t>(lora_row(p.ids, f.place + n * 8 + g, p.rows)) : -1;
    x[n] = static_cast<const T*>(p.in) + (my_row[n] >= 0 ? my_row[n] : 0) * p.ld_in;
  }

  // ---- first product: blocks of 32 k, warp by warp ----
  const int64_t blocks = (p.d_in + 31) / 32;
  const int64_t block0 = blocks * rank >> s_log, block1 = blocks * (rank + 1) >> s_log;
  float acc[RT][NT][4];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][n][i] = 0.f;
  constexpr int kAhead = RT <= 2 && NT <= 2 ? 2 : 1;
  for (int64_t blk = block0 + warp; blk < block1; blk += kAhead * kFewWarps) {
    uint4 xv[kAhead][NT], av[kAhead][RT][2];
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
#pragma unroll
      for (int n = 0; n < NT; ++n) xv[u][n] = load16(x[n] + (in ? k : 0), in && my_row[n] >= 0);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (n >= groups) continue;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const uint4 lo = av[u][t][0], hi = av[u][t][1];
          mma16816<T>(acc[t][n], lo.x, hi.x, lo.y, hi.y, xv[u][n].x, xv[u][n].y);
          mma16816<T>(acc[t][n], lo.z, hi.z, lo.w, hi.w, xv[u][n].z, xv[u][n].w);
        }
      }
  }
  // the warps' sums: the upper ones leave theirs where the lower ones add their own, until kSums are left
  const auto sum_at = [&](int w, int t, int n, int i) {
    return reinterpret_cast<float2*>(warp_sum + w * C::kElems + (t * 16 + g + 8 * i) * C::kRows + n * 8 + 2 * s4);
  };
#pragma unroll
  for (int from = kFewWarps - C::kSums; from >= 0; from -= C::kSums) {
    if (warp >= from && warp < from + C::kSums) {
      const int w = warp - from;
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float2* at = sum_at(w, t, n, i);
            const float2 other = from < kFewWarps - C::kSums ? *at : make_float2(0.f, 0.f);
            *at = make_float2(acc[t][n][2 * i] + other.x, acc[t][n][2 * i + 1] + other.y);
          }
    }
    if (from > 0) __syncthreads();
  }
  if (S > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // (the others have begun)
  __syncthreads();
  // every CTA's sums to all of the cluster's
  for (int e = threadIdx.x * 4; e < C::kElems; e += kFewThreads * 4) {
    float4 v = *reinterpret_cast<const float4*>(warp_sum + e);
#pragma unroll
    for (int w = 1; w < C::kSums; ++w) {
      const float4 o = *reinterpret_cast<const float4*>(warp_sum + w * C::kElems + e);
      v.x += o.x;
      v.y += o.y;
      v.z += o.z;
      v.w += o.w;
    }
    const uint32_t at = smem_u32(part_sum + rank * C::kElems + e);
    for (int c = 0; c < S; ++c)
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_map_shared(at, c)), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
                   : "memory");
  }
  if (S > 1) cluster_sync();
  else __syncthreads();
  // the inner vectors, added up by all threads over the first CTA's sums
  for (int e = threadIdx.x * 4; e < C::kElems; e += kFewThreads * 4) {
    float4 part[kFewCluster];
#pragma unroll
    for (int c = 0; c < kFewCluster; ++c)
      if (c < S) part[c] = *reinterpret_cast<const float4*>(part_sum + c * C::kElems + e);
    float4 v = part[0];
#pragma unroll
    for (int c = 1; c < kFewCluster; ++c)
      if (c < S) {
        v.x += part[c].x;
        v.y += part[c].y;
        v.z += part[c].z;
        v.w += part[c].w;
      }
    *reinterpret_cast<float4*>(part_sum + e) = v;
  }
  __syncthreads();
  // and from them the second product's operand: warp n makes group n's; lane (g, s4) has row g and the ranks r * 32 + s4 * 8 .. + 7
  // of every block r
  if (warp < groups) {
    const int n = warp;
    const int32_t row = n * 8 + g < f.count ? static_cast<int32_t>(lora_row(p.ids, f.place + n * 8 + g, p.rows)) : -1;
    float v[C::kBlocks][8], most = 0.f;
#pragma unroll
    for (int r = 0; r < C::kBlocks; ++r)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = r * 32 + s4 * 8 + i;
        v[r][i] = j < C::kRanks ? part_sum[j * C::kRows + n * 8 + g] : 0.f;
        most = fmaxf(most, fabsf(v[r][i]));
      }
    if (p.inner != nullptr && slot == 0 && row >= 0)
#pragma unroll
      for (int r = 0; r < C::kBlocks; ++r)
#pragma unroll
        for (int i = 0; i < 8; i += 4)
          if (r * 32 + s4 * 8 + i < p.rank)
            *reinterpret_cast<float4*>(p.inner + static_cast<int64_t>(row) * p.rank + r * 32 + s4 * 8 + i) =
                make_float4(v[r][i], v[r][i + 1], v[r][i + 2], v[r][i + 3]);
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    float down, up;
    row_scale<T>(most, &down, &up);
    if (s4 == 0) ups[n * 8 + g] = up;
#pragma unroll
    for (int r = 0; r < C::kBlocks; ++r) {
      uint32_t w[4][kParts];
#pragma unroll
      for (int i = 0; i < 4; ++i) split<T>(v[r][2 * i] * down, v[r][2 * i + 1] * down, w[i]);
#pragma unroll
      for (int q = 0; q < kParts; ++q)
        frag[((n * C::kBlocks + r) * kParts + q) * 32 + lane] = make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]);
    }
  }
  __syncthreads();

  // ---- second product: B's rows n .. n + 7 in this lane, then group by group; the lane's outputs are of the rows 2 s4, 2 s4 + 1 ----
  for (int64_t unit = unit0 + warp; unit < unit1; unit += kFewWarps) {
    const int64_t col = unit * kUnit + g * 8;
    const bool in = col < p.d_out;
    uint4 w[C::kBlocks][8];
#pragma unroll
    for (int r = 0; r < C::kBlocks; ++r) {
      const int j = r * 32 + s4 * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool take = in && j < p.rank;
        w[r][i] = load16(b + (take ? (col + i) * p.rank + j : 0), take);
      }
    }
    uint4 y0[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int32_t to = __shfl_sync(0xffffffffu, my_row[n], (2 * s4 + i) * 4);
        y0[n][i] = to >= 0 && in ? *reinterpret_cast<const uint4*>(static_cast<const T*>(p.base) + to * p.ld_base + col)
                                 : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (n >= groups) break;
      float d[4][4];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) d[t][i] = 0.f;
#pragma unroll
      for (int q = kParts - 1; q >= 0; --q) {
#pragma unroll
        for (int r = 0; r < C::kBlocks; ++r) {
          const uint4 h = frag[((n * C::kBlocks + r) * kParts + q) * 32 + lane];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint4 e = w[r][2 * t], o = w[r][2 * t + 1];
            mma16816<T>(d[t], e.x, o.x, e.y, o.y, h.x, h.y);
            mma16816<T>(d[t], e.z, o.z, e.w, o.w, h.z, h.w);
          }
        }
        if (kLowUp<T> > 0 && q > 0) {
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) d[t][i] *= 1.f / (1 << kLowUp<T>);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int32_t to = __shfl_sync(0xffffffffu, my_row[n], (2 * s4 + i) * 4);
        if (to < 0 || !in) continue;
        const float c = scale * ups[n * 8 + 2 * s4 + i];
        uint32_t y[4] = {y0[n][i].x, y0[n][i].y, y0[n][i].z, y0[n][i].w};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const float2 v = Pair<T>::unpack(y[t]);
          y[t] = Pair<T>::pack(fmaf(c, d[t][i], v.x), fmaf(c, d[t][2 + i], v.y));
        }
        *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + to * p.ld_out + col) = make_uint4(y[0], y[1], y[2], y[3]);
      }
    }
  }
}

template <typename T, int RT, int NT>
ks_status_t launch_few(const char* where, const LoraPass& p, cudaStream_t stream) {
  using C = FewCfg<T, RT, NT>;
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 0 && dev < 64 && !done[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(lora_few_kernel<T, RT, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
      if (e != cudaSuccess) return cuda_status(e, where);
      done[dev] = true;
    }
  }
  const int64_t items = lora_tile_bound(p.rows, p.adapters, C::kRows);
  const int64_t room = static_cast<int64_t>(sm_count()) * 2;
  int s = 3;   // logarithms
  static_assert(kFewCluster == 8, "");
  while (s > 0 && p.d_in < 64 << s) --s;
  // several clusters per item while SMs are idle and the second product is still the larger part of each
  int parts = 0;
  while (items << (s + parts + 1) <= room && p.d_out >= p.d_in << (parts + 1) && p.d_out >= int64_t(kUnit) << (s + parts + 1)) ++parts;
  if (items << (s + parts) > INT32_MAX) KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, std::string(where) + ": grid exceeds CUDA grid limits");
  launch_programmatic_cluster(lora_few_kernel<T, RT, NT>, static_cast<unsigned>(items << (s + parts)), 1u << s, true, kFewThreads,
                              C::kSmem, stream, p, s, parts);
  KSB_CHECK_LAUNCH(where);
  return KS_SUCCESS;
}

template <typename T, int RT>
ks_status_t launch_few_groups(const char* where, const LoraPass& p, cudaStream_t stream) {
  // groups of 8 rows per item: as many as an adapter has on average
  const int64_t mean = (p.rows + p.adapters - 1) / p.adapters;
  return mean <= 8 ? launch_few<T, RT, 1>(where, p, stream)
         : mean <= 16 ? launch_few<T, RT, 2>(where, p, stream)
                      : launch_few<T, RT, 4>(where, p, stream);
}

template <typename T>
ks_status_t launch_few_ranks(const char* where, const LoraPass& p, cudaStream_t stream) {
  return p.rank <= 16   ? launch_few_groups<T, 1>(where, p, stream)
         : p.rank <= 32 ? launch_few_groups<T, 2>(where, p, stream)
         : p.rank <= 64 ? launch_few_groups<T, 4>(where, p, stream)
                        : launch_few_groups<T, 8>(where, p, stream);
}

}  // namespace

ks_status_t lora_few_pass(const char* where, const LoraPass& p, ks_dtype_t dtype, cudaStream_t stream) {
  return dtype == KS_DTYPE_F16 ? launch_few_ranks<__half>(where, p, stream) : launch_few_ranks<__nv_bfloat16>(where, p, stream);
}

}  // namespace sm100
}  // namespace ksb
