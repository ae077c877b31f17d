// Low-rank adapters on the tensor cores: y = y0 + s V (U x) for rows sorted by adapter, forward and, with the factors'
// roles changed, the gradient of the input.
//
// A tile is up to 128 rows of one adapter, and one cluster of CTAs does both products of it: each CTA multiplies its slice
// of U's columns with the rows' elements there, the partial sums [128 x rank] are added up over distributed shared memory
// (in rank order, so all CTAs hold the same bits), and each CTA gives its slice of the outputs. The
// inner vectors never leave the SM, there is one launch, and while the partial sums are exchanged the rows of y0 and V's
// tiles are already on their way: both phases draw on one ring of shared-memory stages.
//   warps 0-7   epilogue: two threads per row. Partial sums out of tensor memory, exchange, split into 16-bit parts,
//               back into tensor memory as the second product's A operand; then y0 + c D, in the stage that holds y0's tile,
//               and out in 64-byte row segments
//   warps 8-11  producer: cp.async of 16 bytes. Rows are gathered by number, tails come as zeros, and neither
//               needs a tensor map (the smallest calls are bound by the host's path)
//   warp 12     tcgen05.mma: M 128 (rows) x N rank, even and odd chunks into sums of their own (an accumulator is cut off, not rounded,
//               at each step: 2.1e-6 of the inner vector over 4096 columns in one, 1.0e-6 in two), then M 128 x N 64 (outputs) with K = rank for each part, the small ones first
// Bound by memory: rows * (d_in + 2 d_out) elements are moved, 2 rank operations for each; the legacy tensor path would be the bound
// from rank 32 on.
#include <algorithm>
#include <mutex>
#include <string>

#include "lora_tiles.cuh"
#include "sm100_lora.cuh"
#include "sm100_host.cuh"
#include "sm100_ptx.cuh"

namespace ksb {
namespace sm100 {
namespace {

constexpr int kTile = kLoraTile;
constexpr int kChunk = 64;                         // columns of a stage: 128 bytes
constexpr int kRowsBytes = kTile * kChunk * 2;     // rows' part of a stage
constexpr int kBlockBytes = 64 * kChunk * 2;       // 64 rows x 128 bytes of a factor
constexpr int kProdWarps = 4;
constexpr int kProdThreads = kProdWarps * 32;
constexpr int kMaxCluster = 8;

// RC: 0 rank <= 32, 1 rank <= 64, 2 rank <= 128. Two CTAs per SM up to rank 64 (one's epilogue under the other's copies).
template <int RC>
struct TileCfg {
  static constexpr int kRanks = 32 << RC;
  static constexpr int RB = RC == 2 ? 2 : 1;           // 64-rank blocks
  static constexpr int kStages = RC == 1 ? 3 : 4;
  static constexpr int kEpiWarps = 8, kMmaWarp = kEpiWarps + kProdWarps;
  static constexpr int kThreads = (kMmaWarp + 1) * 32;
  static constexpr int kStageBytes = kRowsBytes + RB * kBlockBytes;
  static constexpr int kExchange = kTile * kRanks * 4;
  static constexpr int kInner = 2 * kChunk;            // tensor memory: two output buffers, the inner vectors' parts;
  static constexpr int kInnerCols = 32 * RB;           // the sums lie where the outputs come once they are split
  static constexpr int kTmemCols = RB == 1 ? 256 : 512;
  static constexpr int kPerSm = RB == 1 ? 2 : 1;
  static constexpr int kOdd = RB == 1 ? 64 : 384;      // the sums of the odd chunks
  static_assert(64 * RB <= kInner && kInner + 3 * kInnerCols <= (RB == 1 ? kTmemCols : kOdd), "tensor memory layout");
  static constexpr int kBars = 3 * kStages + 8;
  static constexpr int kSmem = kStages * kStageBytes + kExchange + kTile * 4 + 8 * kBars + 64;
  static_assert(kPerSm * (kSmem + 1024) <= 233472, "shared memory");
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// What copies and stores wrote to shared memory before this point, for the tensor cores to read behind it.
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Arrives on the barrier once all copies that this thread has issued are complete. (The barrier counts the arrival; the thread
// that lets the tensor cores read the stage runs fence_async_shared() behind its wait. A producer that waits for its copies
// itself, to place the fence, holds up the next stage's: 113 us against 84 for 16384 rows beside 4096 x 4096, rank 64.)
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// Arrives on the barrier at the same place in the cluster's CTA `rank`; orders this thread's earlier writes.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar, uint32_t rank) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_map_shared(bar, rank)) : "memory");
}
__device__ __forceinline__ bool mbar_wait_cluster(const WaitCtx& ctx, uint32_t bar, uint32_t parity, uint32_t code) {
  const auto done = [&] {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
  };
  const unsigned long long t0 = global_ns();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 256; ++i)
      if (done()) return true;
    if (ctx.raised()) return false;
    if (global_ns() - t0 > kWaitLimitNs) {
      ctx.give_up(code);
      return false;
    }
  }
}
__device__ __forceinline__ void st_shared_cluster_f4(uint32_t addr, const float4& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
// Lane i of the warp writes 8 consecutive columns of tensor memory lane (taddr.lane + i).
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
constexpr float kInf = __builtin_huge_valf();
// The largest of the warp's first values and the smallest of the second.
__device__ __forceinline__ float2 warp_range(float most, float least) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
  }
  return make_float2(most, least);
}

// Whether `ok` (the same for a warp) holds for both warps that share the named barrier `id`. Bounded waits end each on its own, so two
// warps that meet at a barrier settle there whether both go on: one that left alone would leave the other at it for good.
__device__ __forceinline__ bool pair_agrees(uint32_t id, bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "bar.red.and.pred q, %1, 64, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(all)
      : "r"(id), "r"(ok ? 1u : 0u)
      : "memory");
  return all != 0u;
}

struct TileParams {
  LoraPass p;
  unsigned int* fault_word;
  uint32_t idesc1, idesc2;
  int rank16;       // rank rounded up to 16
  int cluster_log;  // CTAs of a cluster: 1 << cluster_log
  int in_chunks, out_chunks;
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// CTA `rank` of S adds up its part of the cluster's sums, in rank order, and writes the totals back to all of them, where only it has
// read. Piece e is the 16 bytes of row e % rows and four ranks. A thread has eight loads from other SMs in flight.
template <int S, int THREADS>
__device__ __forceinline__ void reduce_scatter(uint32_t exchange, int pieces, int quarters, int rank) {
  constexpr int kAtOnce = kMaxCluster / S;
  const int end = pieces / S * (rank + 1);
  for (int e0 = pieces / S * rank + threadIdx.x; e0 < end; e0 += kAtOnce * THREADS) {
    float4 part[kAtOnce][S];
    uint32_t at[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int e = e0 + u * THREADS, j = (e >> 5) / quarters, row = e - j * quarters * 32;
      at[u] = exchange + (j * kTile + row) * 16;
#pragma unroll
      for (int c = 0; c < S; ++c)
        if (e < end) part[u][c] = ld_shared_cluster_f4(cluster_map_shared(at[u], c));
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (e0 + u * THREADS >= end) continue;
      float4 sum = part[u][0];
#pragma unroll
      for (int c = 1; c < S; ++c) {
        sum.x += part[u][c].x;
        sum.y += part[u][c].y;
        sum.z += part[u][c].z;
        sum.w += part[u][c].w;
      }
#pragma unroll
      for (int c = 0; c < S; ++c) st_shared_cluster_f4(cluster_map_shared(at[u], c), sum);
    }
  }
}

template <typename T, int RC, bool FWD>
__global__ void __launch_bounds__(TileCfg<RC>::kThreads, TileCfg<RC>::kPerSm) lora_tile_kernel(const __grid_constant__ TileParams q) {
  using C = TileCfg<RC>;
  constexpr int RB = C::RB, kParts = kInnerParts<T>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const LoraPass& p = q.p;
  const uint32_t ring = smem_u32(smem);   // (1024-byte aligned: there is no static shared memory)
  const uint32_t exchange = ring + C::kStages * C::kStageBytes;
  int32_t* row_of = reinterpret_cast<int32_t*>(smem + C::kStages * C::kStageBytes + C::kExchange);
  uint64_t* bar_mem = reinterpret_cast<uint64_t*>(row_of + kTile);
  const uint32_t bars = smem_u32(bar_mem);
  const auto full = [&](int s) { return bars + 8u * s; };                       // copies have landed
  const auto free1 = [&](int s) { return bars + 8u * (C::kStages + s); };       // first product has read the stage
  const auto free2 = [&](int s) { return bars + 8u * (2 * C::kStages + s); };   // the epilogue has written it out
  const uint32_t bar_sums = bars + 8u * (3 * C::kStages);        // first product complete
  const uint32_t bar_inner = bar_sums + 8;                       // second product's operand is in tensor memory
  const uint32_t bar_parts = bar_sums + 16;                      // the cluster's partial sums are in shared memory
  const uint32_t bar_total = bar_sums + 24;                      // and so are their totals
  const auto out_full = [&](int b) { return bar_sums + 32u + 8u * b; };
  const auto out_free = [&](int b) { return bar_sums + 48u + 8u * b; };
  volatile uint32_t* words = reinterpret_cast<volatile uint32_t*>(bar_mem + C::kBars);   // tmem address, abort, tile
  const WaitCtx wctx{smem_u32(const_cast<uint32_t*>(words) + 1), q.fault_word};
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int S = 1 << q.cluster_log;
  const uint32_t rank = blockIdx.x & (S - 1);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full(s), kProdThreads);
      mbar_init(free1(s), 1);
      mbar_init(free2(s), C::kEpiWarps);
    }
    mbar_init(bar_sums, 1);
    mbar_init(bar_inner, C::kEpiWarps * 32);
    mbar_init(bar_parts, static_cast<uint32_t>(S) * C::kEpiWarps);
    mbar_init(bar_total, static_cast<uint32_t>(S) * C::kEpiWarps);
    for (int b = 0; b < 2; ++b) {
      mbar_init(out_full(b), 1);
      mbar_init(out_free(b), C::kEpiWarps);
    }
    words[1] = 0u;
    fence_barrier_init();
  }
  __syncwarp();
  bool joined = S == 1;            // (waited for the other CTAs' barriers to be initialised)
  if (!joined) cluster_arrive();
  grid_dependency_wait();
  if (warp == C::kMmaWarp) {   // (behind the wait: a kernel that still runs may need the columns)
    tmem_alloc(smem_u32(const_cast<uint32_t*>(words)), C::kTmemCols);
    tmem_relinquish();
  }
  if (warp == 0) {
    const TilePlace f = find_tile<kTile>(p.offsets, p.adapters, p.rows, blockIdx.x >> q.cluster_log);
    if (lane == 0) {
      words[2] = static_cast<uint32_t>(f.adapter);
      words[3] = static_cast<uint32_t>(f.count);
      words[4] = static_cast<uint32_t>(f.place);
    }
#pragma unroll
    for (int i = 0; i < kTile / 32; ++i) {
      const int r = i * 32 + lane;
      row_of[r] = r < f.count ? static_cast<int32_t>(lora_row(p.ids, f.place + r, p.rows)) : -1;
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = words[0];
  const int adapter = static_cast<int>(words[2]);
  const int count = static_cast<int>(words[3]);
  const int64_t place = words[4];

  // this CTA's 64-column chunks of the inputs and of the outputs
  const auto share = [&](int chunks, uint32_t r) { return static_cast<int>((static_cast<uint32_t>(chunks) * r) >> q.cluster_log); };
  const int in0 = share(q.in_chunks, rank), n1 = share(q.in_chunks, rank + 1) - in0;
  const int out0 = share(q.out_chunks, rank), n2 = share(q.out_chunks, rank + 1) - out0;
  const int quarters = (count + 31) / 32;   // of the tile that hold rows

  if (adapter == p.adapters) {
    // rows without an adapter: y = y0
    if (p.out != p.base) {
      const int64_t c0 = static_cast<int64_t>(out0) * kChunk;
      const int64_t c1 = min(p.d_out, c0 + static_cast<int64_t>(n2) * kChunk);
      for (int r = warp; r < count; r += C::kThreads / 32) {
        const int64_t row = row_of[r];
        if (row < 0) continue;
        const T* src = static_cast<const T*>(p.base) + row * p.ld_base;
        T* dst = static_cast<T*>(p.out) + row * p.ld_out;
        for (int64_t c = c0 + lane * 8; c < c1; c += 8 * 256) {
          uint4 v[8];
#pragma unroll
          for (int u = 0; u < 8; ++u)
            if (c + u * 256 < c1) v[u] = *reinterpret_cast<const uint4*>(src + c + u * 256);
#pragma unroll
          for (int u = 0; u < 8; ++u)
            if (c + u * 256 < c1) __stcs(reinterpret_cast<uint4*>(dst + c + u * 256), v[u]);
        }
      }
    }
  } else if (adapter >= 0) {
    const int total = n1 + n2;
    if (warp >= C::kEpiWarps && warp < C::kMmaWarp) {
      // ---- producer ----
      const int t = threadIdx.x - C::kEpiWarps * 32;
      const int c8 = t & 7, r0 = t >> 3;                         // rows' part: 16 bytes of the rows r0 + 16 i
      const int j8 = t % (8 * RB), i0 = t / (8 * RB);            // 64 rows of `rank` columns: rows i0 + 16 / RB * i
      const T* u = static_cast<const T*>(p.u) + static_cast<int64_t>(adapter) * p.rank * p.d_in;
      const T* v = static_cast<const T*>(p.v) + static_cast<int64_t>(adapter) * p.rank * p.d_out;
      const T* src[8];
      uint32_t have = 0u;
      const auto aim = [&](const void* m, int64_t ld, int chunk) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int32_t row = row_of[r0 + 16 * i];
          if (row >= 0) have |= 1u << i;
          src[i] = static_cast<const T*>(m) + (row >= 0 ? row : 0) * ld + static_cast<int64_t>(chunk) * kChunk + c8 * 8;
        }
      };
      aim(p.in, p.ld_in, in0);
#pragma unroll 1
      for (int it = 0; it < total; ++it) {
        const int s = it % C::kStages;
        const int before = it - C::kStages;   // the stage's last use
        if (before >= 0) {
          const int n2_before = before - n1;
          const uint32_t bar = n2_before < 0 ? free1(s) : free2(s);
          const uint32_t parity = (n2_before < 0 ? before / C::kStages : n2_before / C::kStages) & 1;
          if (!mbar_wait(wctx, bar, parity, 0x31)) break;
        }
        if (it == n1) aim(p.base, p.ld_base, out0);
        const bool one = it < n1;
        const int64_t col = static_cast<int64_t>(one ? in0 + it : out0 + it - n1) * kChunk;
        const int64_t width = one ? p.d_in : p.d_out;
        const uint32_t dst = ring + s * C::kStageBytes;
        const bool in_width = col + c8 * 8 < width;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          // (places without a row are cleared once; what the epilogue leaves there is zero again)
          const bool row = have >> i & 1u;
          if (row || it < C::kStages)
            cp_async16(dst + r0 * 128 + ((c8 ^ (r0 & 7)) << 4) + i * 2048, row && in_width ? src[i] : p.in, row && in_width);
          src[i] += kChunk;
        }
        const uint32_t wdst = dst + kRowsBytes;
        const T* w = one ? u : v;
        if (one == FWD) {
          // rank rows of 64 columns, `width` apart
          const T* from = w + r0 * width + col + c8 * 8;
#pragma unroll
          for (int i = 0; i < 4 * RB; ++i) {
            const int j = r0 + 16 * i;
            const bool take = in_width && j < p.rank;
            if (i * 16 < q.rank16)
              cp_async16(wdst + r0 * 128 + ((c8 ^ (r0 & 7)) << 4) + i * 2048, take ? from + i * 16 * width : p.u, take);
          }
        } else if (j8 * 8 < q.rank16) {
          // 64 rows of `rank` columns
          const T* from = w + (col + i0) * p.rank + j8 * 8;
#pragma unroll
          for (int i = 0; i < 4 * RB; ++i) {
            const int r = i0 + 16 / RB * i;
            const bool take = col + r < width && j8 * 8 < p.rank;
            cp_async16(wdst + (j8 >> 3) * kBlockBytes + r * 128 + (((j8 & 7) ^ (r & 7)) << 4),
                       take ? from + static_cast<int64_t>(16 / RB * i) * p.rank : p.u, take);
          }
        }
        cp_async_arrive(full(s));
      }
      cp_async_wait_all();
    } else if (warp == C::kMmaWarp) {
      // ---- tensor cores ----
      bool ok = true;
      for (int it = 0; it < n1; ++it) {
        const int s = it % C::kStages;
        if (!(ok = all_lanes(mbar_wait(wctx, full(s), (it / C::kStages) & 1, 0x33)))) break;
        fence_async_shared();
        tc_fence_after_sync();
        const uint32_t a = ring + s * C::kStageBytes, b = a + kRowsBytes;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const uint64_t ad = umma_smem_desc_sw128(a + kk * 32, 16, 1024);
          const uint64_t bd = FWD ? umma_smem_desc_sw128(b + kk * 32, 16, 1024)
                                  : umma_smem_desc_sw128(b + kk * 16 * 128, kBlockBytes, 1024);
          umma_f16_elect(tmem + (it & 1 ? C::kOdd : 0), ad, bd, q.idesc1, it > 1 || kk > 0 ? 1u : 0u);
        }
        tc_commit_elect(free1(s));
      }
      if (ok && n1 > 0) tc_commit_elect(bar_sums);
      if (ok && n2 > 0) ok = all_lanes(mbar_wait_long(wctx, bar_inner, 0, 0x34));
      tc_fence_after_sync();
      for (int j = 0; ok && j < n2; ++j) {
        const int it = n1 + j, s = it % C::kStages, b = j & 1;
        if (j >= 2 && !(ok = all_lanes(mbar_wait(wctx, out_free(b), ((j >> 1) - 1) & 1, 0x35)))) break;
        if (!(ok = all_lanes(mbar_wait(wctx, full(s), (it / C::kStages) & 1, 0x36)))) break;
        fence_async_shared();
        tc_fence_after_sync();
        const uint32_t w = ring + s * C::kStageBytes + kRowsBytes;
        const uint32_t d = tmem + b * kChunk;
#pragma unroll
        for (int part = kParts - 1; part >= 0; --part)
          for (int kk = 0; kk < q.rank16 / 16; ++kk) {
            const uint64_t bd = FWD ? umma_smem_desc_sw128(w + (kk >> 2) * kBlockBytes + (kk & 3) * 32, 16, 1024)
                                    : umma_smem_desc_sw128(w + kk * 16 * 128, kBlockBytes, 1024);
            const uint32_t inner = tmem + C::kInner + part * C::kInnerCols + kk * 8;
            if (kLowUp<T> > 0 && part == 0 && kk == 0) umma_f16_tmem_a_down_elect<kLowUp<T>>(d, inner, bd, q.idesc2);
            else umma_f16_tmem_a_elect(d, inner, bd, q.idesc2, part < kParts - 1 || kk > 0 ? 1u : 0u);
          }
        tc_commit_elect(out_full(b));
      }
    } else {
      // ---- epilogue: a thread per row and half (of the ranks, of a chunk's columns) ----
      const int quarter = warp & 3, half = warp >> 2;
      const int r = quarter * 32 + lane;
      const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter) << 21);
      const float s = __ldg(p.scales + adapter);
      const int blocks = q.rank16 / 16;
      const bool used = quarter < quarters;   // (the quarters without rows only keep step)
      if (!joined) cluster_wait();
      joined = true;
      bool ok = n1 == 0 || all_lanes(mbar_wait_long(wctx, bar_sums, 0, 0x37));
      tc_fence_after_sync();
      const auto own_sums = [&](int b, uint32_t (&x)[16]) {   // 16 ranks of the row, over this CTA's columns
        tmem_ld(lanes + b * 16, x);
        tmem_wait_ld(x);
        if (n1 > 1) {
          uint32_t odd[16];
          tmem_ld(lanes + C::kOdd + b * 16, odd);
          tmem_wait_ld(odd);
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) + __uint_as_float(odd[i]));
        }
      };
      if (ok && S > 1) {
        // ranks 4 j .. of row r at exchange + (j * 128 + r) * 16
        for (int b = used ? half : blocks; b < blocks; b += 2) {
          uint32_t x[16] = {};
          if (n1 > 0) own_sums(b, x);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            st_shared_v4(exchange + ((b * 4 + i) * kTile + r) * 16, x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        }
        __syncwarp();
        if (lane < S) mbar_arrive_cluster(bar_parts, lane);
        ok = all_lanes(mbar_wait_cluster(wctx, bar_parts, 0, 0x38));
        if (ok) {
          const int pieces = q.rank16 / 4 * quarters * 32;
          if (S == 2) reduce_scatter<2, C::kEpiWarps * 32>(exchange, pieces, quarters, rank);
          else if (S == 4) reduce_scatter<4, C::kEpiWarps * 32>(exchange, pieces, quarters, rank);
          else reduce_scatter<8, C::kEpiWarps * 32>(exchange, pieces, quarters, rank);
          __syncwarp();
          if (lane < S) mbar_arrive_cluster(bar_total, lane);
          ok = all_lanes(mbar_wait_cluster(wctx, bar_total, 0, 0x3b));
        }
      }
      if (used) ok = pair_agrees(1 + quarter, ok);
      if (ok) {
        const auto sums_of = [&](int b, uint32_t (&x)[16]) {
          if (S > 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint4 v = ld_shared_v4(exchange + ((b * 4 + i) * kTile + r) * 16);
              x[4 * i] = v.x;
              x[4 * i + 1] = v.y;
              x[4 * i + 2] = v.z;
              x[4 * i + 3] = v.w;
            }
          } else {
            own_sums(b, x);
          }
        };
        const int32_t row = row_of[r];
        constexpr bool kRanges = std::is_same<T, __half>::value && !FWD;
        float most = 0.f, least = kInf, down, up;
        for (int b = used ? 0 : blocks; b < blocks; ++b) {
          uint32_t x[16];
          sums_of(b, x);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float v = fabsf(__uint_as_float(x[i]));
            most = fmaxf(most, v);
            if (kRanges) least = v > 0.f ? fminf(least, v) : least;
          }
        }
        row_scale<T>(most, &down, &up);
        const float inner_scale = p.scale_inner ? s : 1.f;
        float* inner = p.inner != nullptr && rank == 0 && row >= 0 ? p.inner + static_cast<int64_t>(row) * p.rank : nullptr;
        for (int b = half; b < blocks; b += 2) {
          uint32_t x[16], inner_part[kParts][8];
          if (used) {
            sums_of(b, x);
          } else {   // (rows of zeros, whatever tensor memory held)
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = 0u;
          }
          if (inner != nullptr) {
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              if (b * 16 + i < p.rank)
                *reinterpret_cast<float4*>(inner + b * 16 + i) =
                    make_float4(inner_scale * __uint_as_float(x[i]), inner_scale * __uint_as_float(x[i + 1]),
                                inner_scale * __uint_as_float(x[i + 2]), inner_scale * __uint_as_float(x[i + 3]));
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t w[kParts];
            split<T>(__uint_as_float(x[2 * i]) * down, __uint_as_float(x[2 * i + 1]) * down, w);
#pragma unroll
            for (int part = 0; part < kParts; ++part) inner_part[part][i] = w[part];
          }
#pragma unroll
          for (int part = 0; part < kParts; ++part) tmem_st8(lanes + C::kInner + part * C::kInnerCols + b * 8, inner_part[part]);
        }
        tmem_wait_st();
        tc_fence_before_sync();
        mbar_arrive(bar_inner);
        if (kRanges && p.range_g != nullptr && rank == 0 && half == 0) {
          float most_h = 0.f, least_h = kInf;
          if (row >= 0)
            for (int i = 0; i < p.rank; i += 4) {
              const float4 v = __ldg(reinterpret_cast<const float4*>(p.h + static_cast<int64_t>(row) * p.rank + i));
              const float f[4] = {fabsf(v.x), fabsf(v.y), fabsf(v.z), fabsf(v.w)};
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                most_h = fmaxf(most_h, f[u]);
                least_h = f[u] > 0.f ? fminf(least_h, f[u]) : least_h;
              }
            }
          const float2 range_g = warp_range(row >= 0 ? most * fabsf(inner_scale) : 0.f, row >= 0 ? least * fabsf(inner_scale) : kInf);
          const float2 range_h = warp_range(most_h, least_h);
          if (lane == 0 && quarter * 32 < count) {
            p.range_g[place + quarter * 32] = range_g;
            p.range_h[place + quarter * 32] = range_h;
          }
        }
        // second product: y0 + c D in the stage that holds y0, then out: of the quarter's 32 rows a warp stores 16, 128 bytes of each
        // (each half its 64 bytes: 106 us against 83 for 16384 rows beside 4096 x 4096)
        const float c = s * up;
        const int piece = lane & 7, out_row = quarter * 32 + half * 16 + (lane >> 3);
        T* dst[4];
        uint32_t have = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int32_t to = row_of[out_row + i * 4];
          if (to >= 0) have |= 1u << i;
          dst[i] = static_cast<T*>(p.out) + (to >= 0 ? to : 0) * p.ld_out + static_cast<int64_t>(out0) * kChunk + piece * 8;
        }
#pragma unroll 1
        for (int j = 0; j < n2; ++j) {
          const int it = n1 + j, st = it % C::kStages, b = j & 1;
          const uint32_t tile = ring + st * C::kStageBytes;
          ok = all_lanes(mbar_wait(wctx, full(st), (it / C::kStages) & 1, 0x3a));
          uint4 y[4];
          if (used) {
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = ld_shared_v4(tile + r * 128 + (((half * 4 + i) ^ (r & 7)) << 4));
          }
          ok = ok && all_lanes(mbar_wait(wctx, out_full(b), (j >> 1) & 1, 0x39));
          if (!used && !ok) break;
          tc_fence_after_sync();
          if (used) {
            uint32_t d[32];
            tmem_ld(lanes + b * kChunk + half * 32, d);
            tmem_wait_ld(d);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t w[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float2 f = Pair<T>::unpack(w[k]);
                w[k] = Pair<T>::pack(fmaf(c, __uint_as_float(d[i * 8 + k * 2]), f.x),
                                     fmaf(c, __uint_as_float(d[i * 8 + k * 2 + 1]), f.y));
              }
              st_shared_v4(tile + r * 128 + (((half * 4 + i) ^ (r & 7)) << 4), w[0], w[1], w[2], w[3]);
            }
            tc_fence_before_sync();
            if (!(ok = pair_agrees(1 + quarter, ok))) break;   // (both halves of the quarter's rows are there)
            const bool in_width = static_cast<int64_t>(out0 + j) * kChunk + piece * 8 < p.d_out;
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = ld_shared_v4(tile + (out_row + i * 4) * 128 + ((piece ^ ((out_row + i * 4) & 7)) << 4));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (in_width && (have >> i & 1u)) *reinterpret_cast<uint4*>(dst[i]) = y[i];
              dst[i] += kChunk;
            }
          }
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(out_free(b));
            mbar_arrive(free2(st));
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  if (S > 1) {
    if (!joined) cluster_wait();
    cluster_sync();   // (nobody reads this CTA's partial sums any more)
  } else {
    __syncthreads();
  }
  tc_fence_after_sync();
  if (warp == C::kMmaWarp) tmem_dealloc(tmem, C::kTmemCols);
}

template <typename T, int RC, bool FWD>
ks_status_t launch_tile(const char* where, const TileParams& q, int64_t tiles, cudaStream_t stream) {
  using C = TileCfg<RC>;
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 0 && dev < 64 && !done[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(lora_tile_kernel<T, RC, FWD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
      if (e != cudaSuccess) return cuda_status(e, where);
      done[dev] = true;
    }
  }
  launch_programmatic_cluster(lora_tile_kernel<T, RC, FWD>, static_cast<unsigned>(tiles << q.cluster_log), 1u << q.cluster_log,
                              true, C::kThreads, C::kSmem, stream, q);
  KSB_CHECK_LAUNCH(where);
  return KS_SUCCESS;
}

// ---------------------------------------------------------------------------------
// gradients of the factors
// ---------------------------------------------------------------------------------
// dA^T [k, rank] = sum over the adapter's rows of x_row g_row^T, and dB [n, rank] = s sum dout_row h_row^T: the same product of a
// matrix of 16-bit rows, taken in slabs of 256 columns, with fp32 vectors of `rank` numbers. A cluster of CTAs has a slab of one
// adapter and splits its rows; the parts are added up over distributed shared memory in rank order. Rows are contracted, so both operands
// are stored with the contracted index outside (MN-major), as they lie in memory; a vector is split into 16-bit
// parts, the first parts' sums apart from the others', which are small. In f16 the vectors are scaled by a power of two per adapter, from the ranges that the pass before left; where an adapter's numbers lie
// further apart than the parts can hold (a factor of 2^33) its sums are made once more in fp32, row by row, and so are sums that
// are not finite. (All of d_b for 16384 rows of rank 64 beside 4096 x 4096: 7.6 ms in place of
// 0.15 for the call, which only such numbers pay.)
//   warps 0-7   split vectors (registers, two stages ahead -> shared memory, four warps a stage), at the end the sums
//   warps 8-11  copies of 64 rows x 512 bytes: one TMA load per 128 bytes of width where the rows lie together (a sequence), cp.async where
//               they do not (TMA gathers of four rows: 322 us against 196 for 16384 rows of 3 adapters, rank 16: a copy of 512 bytes takes 40 clocks)
//   warp 12     tcgen05.mma: per stage 2 (128-column halves) x 4 (16 rows each), N = twice the rank (first and second parts side by side, so
//               that the rows are read once for both), and once more with N = rank for the third parts, added to the second's
// Bound by memory: every element of x and dout is read once; the vectors are read again from L2 per slab (half the bytes of
// a slab's rows at rank 64, which is why a slab is as wide as tensor memory and the ring allow two CTAs per SM).
constexpr int kSlab = 256;

template <typename T, int RB>
struct GradCfg {
  static constexpr int kParts = kInnerParts<T>;
  static constexpr int kStages = RB == 1 || kParts == 3 ? 2 : 3;
  static constexpr int kVecWarps = 8, kMmaWarp = kVecWarps + kProdWarps;
  static constexpr int kThreads = (kMmaWarp + 1) * 32;
  static constexpr int kRows = 64 * kSlab * 2;             // four blocks of 64 rows x 128 bytes
  static constexpr int kPart = RB * kBlockBytes;           // one 16-bit part of the vectors: 64 RB columns
  static constexpr int kStageBytes = kRows + kParts * kPart;
  static constexpr int kHalf = 128 * RB;                   // tensor memory of a half: the sums of the first parts and of the others
  static constexpr int kTmemCols = 2 * kHalf;
  static constexpr int kPerSm = RB == 1 ? 2 : 1;
  static constexpr int kBars = 3 * kStages + 1;
  static constexpr int kSums = kSlab * 64 * RB * 4;        // over the ring, once it is drained
  static_assert(kSums <= kStages * kStageBytes, "the sums lie over the ring");
  static constexpr int kSmem = kStages * kStageBytes + 8 * kBars + 64;
  static_assert(kPerSm * (kSmem + 1024) <= 233472, "shared memory");
};

struct GradParams {
  LoraWeightGrad p;
  unsigned int* fault_word;
  uint32_t idesc2, idesc1;   // N = twice the rank, the rank
  int rank16, cluster_log;   // CTAs of a cluster: 1 << cluster_log
  int slabs_a, slabs;     // slabs of x, of both
};

// Adds up the S parts [rank16][256 / S] fp32 of a share of a slab's columns at `sums`, in order, and writes them, 8 numbers that lie
// together in the result at a time.
template <typename T, int S, int THREADS>
__device__ __forceinline__ void add_parts(const LoraWeightGrad& p, uint32_t sums, int rank16, bool is_a, int adapter, int64_t col0) {
  constexpr int kCols = kSlab / S;
  const int64_t width = is_a ? p.k : p.n;
  T* out = static_cast<T*>(is_a ? p.d_a : p.d_b) + static_cast<int64_t>(adapter) * p.rank * width;
  const int items = p.rank * kCols / 8;
  for (int e = threadIdx.x; e < items; e += THREADS) {
    // 8 columns of a rank, or 8 ranks of a column
    const int j = is_a ? e / (kCols / 8) : e / kCols * 8, m = is_a ? e % (kCols / 8) * 8 : e % kCols;
    if (col0 + m >= width) continue;
    float v[8] = {};
#pragma unroll
    for (int c = 0; c < S; ++c) {
      const uint32_t at = sums + ((c * rank16 + j) * kCols + m) * 4;
      if (is_a) {
        const uint4 x = ld_shared_v4(at), y = ld_shared_v4(at + 16);
        const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += __uint_as_float(w[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += ld_shared_f32(at + i * kCols * 4);
      }
    }
    *reinterpret_cast<uint4*>(out + (is_a ? j * width + col0 + m : (col0 + m) * p.rank + j)) =
        make_uint4(Pair<T>::pack(v[0], v[1]), Pair<T>::pack(v[2], v[3]), Pair<T>::pack(v[4], v[5]), Pair<T>::pack(v[6], v[7]));
  }
}

// The sums of the places [first, last) for a column and the ranks j .. j + 3, in fp32, row by row.
template <typename T>
__device__ __forceinline__ float4 plain_sums(const LoraWeightGrad& p, bool is_a, int64_t first, int64_t last, int64_t col, int j) {
  const T* m = static_cast<const T*>(is_a ? p.x : p.d_out) + col;
  const int64_t ld = is_a ? p.ld_x : p.ld_d_out;
  const float* vecs = (is_a ? p.g : p.h) + j;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int kAhead = 4;   // rows asked for at a time, without branches between the loads
#pragma unroll 1
  for (int64_t place = first; place < last; place += kAhead) {
    int32_t row[kAhead];
    T x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) row[u] = static_cast<int32_t>(lora_row(p.ids, place + u < last ? place + u : last - 1, p.rows));
#pragma unroll
    for (int u = 0; u < kAhead; ++u) x[u] = m[(row[u] >= 0 ? row[u] : 0) * ld];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(vecs + static_cast<int64_t>(row[u] >= 0 ? row[u] : 0) * p.rank));
      const bool take = row[u] >= 0 && place + u < last;
      const float f = to_f32<T>(x[u]);
      sum.x = take ? fmaf(v.x, f, sum.x) : sum.x;
      sum.y = take ? fmaf(v.y, f, sum.y) : sum.y;
      sum.z = take ? fmaf(v.z, f, sum.z) : sum.z;
      sum.w = take ? fmaf(v.w, f, sum.w) : sum.w;
    }
  }
  return sum;
}

template <typename T, int RB>
__global__ void __launch_bounds__(GradCfg<T, RB>::kThreads, GradCfg<T, RB>::kPerSm) lora_weight_grad_kernel(const __grid_constant__ GradParams q,
                                                                                                       const __grid_constant__ CUtensorMap map_x,
                                                                                                       const __grid_constant__ CUtensorMap map_d_out) {
  using C = GradCfg<T, RB>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const LoraWeightGrad& p = q.p;
  const uint32_t ring = smem_u32(smem);   // (1024-byte aligned: there is no static shared memory)
  uint64_t* bar_mem = reinterpret_cast<uint64_t*>(smem + C::kStages * C::kStageBytes);
  const uint32_t bars = smem_u32(bar_mem);
  const auto full = [&](int s) { return bars + 8u * s; };   // the vectors are there, and rows that were copied one by one
  const auto freed = [&](int s) { return bars + 8u * (C::kStages + s); };
  const auto landed = [&](int s) { return bars + 8u * (2 * C::kStages + s); };   // and rows by TMA
  const uint32_t bar_sums = bars + 8u * (3 * C::kStages);
  volatile uint32_t* words = reinterpret_cast<volatile uint32_t*>(bar_mem + C::kBars);
  const WaitCtx wctx{smem_u32(const_cast<uint32_t*>(words) + 1), q.fault_word};
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int S = 1 << q.cluster_log;
  const int rank = blockIdx.x & (S - 1);
  const int item = blockIdx.x >> q.cluster_log;
  const int adapter = item / q.slabs;
  const int slab = item - adapter * q.slabs;
  const bool is_a = slab < q.slabs_a;
  const int64_t col0 = static_cast<int64_t>(is_a ? slab : slab - q.slabs_a) * kSlab;
  const int64_t width = is_a ? p.k : p.n;
  const float* vecs = is_a ? p.g : p.h;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full(s), C::kVecWarps / 2 * 32 + kProdThreads);
      mbar_init(freed(s), 1);
      mbar_init(landed(s), 1);
    }
    mbar_init(bar_sums, 1);
    words[1] = 0u;
    fence_barrier_init();
  }
  grid_dependency_wait();
  if (warp == C::kMmaWarp) {   // (behind the wait: a kernel that still runs may need the columns)
    tmem_alloc(smem_u32(const_cast<uint32_t*>(words)), C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = words[0];
  const int64_t begin = lora_offset(p.offsets, adapter, p.rows);
  const int64_t count = max(lora_offset(p.offsets, adapter + 1, p.rows) - begin, int64_t(0));
  const int64_t chunks = (count + 63) / 64;
  const int64_t chunk0 = chunks * rank >> q.cluster_log;
  const int n = static_cast<int>((chunks * (rank + 1) >> q.cluster_log) - chunk0);
  const auto row_at = [&](int64_t chunk, int i) -> int32_t {   // row i of a chunk, -1 past the end
    const int64_t at = chunk * 64 + i;
    return at < count ? static_cast<int32_t>(lora_row(p.ids, begin + at, p.rows)) : -1;
  };
  float up = 1.f;
  bool far = false;

  if (warp >= C::kVecWarps && warp < C::kMmaWarp) {
    // ---- copies. 64 rows that lie together come by TMA; others one by one: a warp takes every fourth, a lane 16 bytes of it ----
    const int w = warp - C::kVecWarps;
    const int64_t ld = is_a ? p.ld_x : p.ld_d_out;
    const T* rows = static_cast<const T*>(is_a ? p.x : p.d_out);
    const int64_t col = col0 + lane * 8;
    const bool in_width = col < width;
    const T* src = rows + (in_width ? col : 0);
    const uint32_t dst0 = ring + (lane >> 3) * kBlockBytes + w * 128;
    // (row w + 4 i: its swizzle is (w + 4 i) & 7)
    const uint32_t even = ((lane & 7) ^ w) << 4, odd = ((lane & 7) ^ (w + 4)) << 4;
    int32_t lo = n > 0 ? row_at(chunk0, lane) : -1, hi = n > 0 ? row_at(chunk0, lane + 32) : -1;   // the chunk's rows
    int it = 0;
    bool ok = true;
#pragma unroll 1
    for (; it < n; ++it) {
      const int s = it % C::kStages;
      if (it >= C::kStages && !(ok = all_lanes(mbar_wait(wctx, freed(s), (it / C::kStages - 1) & 1, 0x41)))) break;
      const int32_t row0 = __shfl_sync(0xffffffffu, lo, 0), now_lo = lo, now_hi = hi;
      const bool together = __all_sync(0xffffffffu, lo >= 0 && lo == row0 + lane && hi == row0 + 32 + lane);
      if (it + 1 < n) {
        lo = row_at(chunk0 + it + 1, lane);
        hi = row_at(chunk0 + it + 1, lane + 32);
      }
      const uint32_t dst = ring + s * C::kStageBytes;
      if (together) {
        if (w == 0 && lane == 0) {
          mbar_arrive_expect_tx(landed(s), C::kRows);
#pragma unroll
          for (int i = 0; i < kSlab / 64; ++i)
            tma_load_2d(dst + i * kBlockBytes, is_a ? &map_x : &map_d_out, landed(s), static_cast<int>(col0) + i * 64, row0);
        }
        mbar_arrive(full(s));
        continue;
      }
      if (w == 0 && lane == 0) mbar_arrive(landed(s));
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int32_t row = __shfl_sync(0xffffffffu, i < 8 ? now_lo : now_hi, (w + 4 * i) & 31);
        const bool take = in_width && row >= 0;
        cp_async16(dst0 + s * C::kStageBytes + i * 512 + (i & 1 ? odd : even), take ? src + row * ld : rows, take);
      }
      cp_async_arrive(full(s));
    }
    cp_async_wait_all();
    if (!ok)   // (and for copies by TMA)
      for (int i = it - C::kStages; i < it; ++i) mbar_wait(wctx, landed(i % C::kStages), (i / C::kStages) & 1, 0x45);
  } else if (warp < C::kVecWarps) {
    // ---- vectors: the two halves of the warps take the chunks in turn, a thread 8 ranks of every (16 / RB)-th row ----
    const int turn = warp / (C::kVecWarps / 2), t = threadIdx.x % (C::kVecWarps * 16);
    const int c8 = t % (8 * RB), r0 = t / (8 * RB);
    constexpr int kStep = 16 / RB, kMine = 64 / kStep;
    const bool used = c8 * 8 < q.rank16, has = c8 * 8 < p.rank;
    float down = 1.f;
    if (std::is_same<T, __half>::value) {
      const float2* ranges = is_a ? p.range_g : p.range_h;
      float2 r = make_float2(0.f, kInf);
      for (int64_t i = lane; i * 32 < count; i += 32) {
        const float2 v = __ldg(ranges + begin + i * 32);
        r = make_float2(fmaxf(r.x, v.x), fminf(r.y, v.y));
      }
      r = warp_range(r.x, r.y);
      row_scale<T>(r.x, &down, &up);
      far = far_apart(r.x, r.y);
    }
    int32_t row[kMine];
    float4 v[kMine][2];
    const auto find = [&](int64_t chunk) {
#pragma unroll
      for (int i = 0; i < kMine; ++i) row[i] = used ? row_at(chunk, r0 + i * kStep) : -1;
    };
    const auto load = [&] {
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const bool take = has && row[i] >= 0;
        const float4* from = reinterpret_cast<const float4*>(vecs + static_cast<int64_t>(take ? row[i] : 0) * p.rank + (take ? c8 * 8 : 0));
        v[i][0] = take ? __ldg(from) : make_float4(0.f, 0.f, 0.f, 0.f);
        v[i][1] = take ? __ldg(from + 1) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    };
    bool ok = true;
    if (turn < n) {
      find(chunk0 + turn);
      load();
      if (turn + 2 < n) find(chunk0 + turn + 2);
    }
#pragma unroll 1
    for (int it = turn; it < n; it += 2) {
      const int s = it % C::kStages;
      if (it >= C::kStages && !(ok = mbar_wait(wctx, freed(s), (it / C::kStages - 1) & 1, 0x42))) break;
      const uint32_t dst = ring + s * C::kStageBytes + C::kRows;
      if (used) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const int r = r0 + i * kStep;
          const float f[8] = {v[i][0].x * down, v[i][0].y * down, v[i][0].z * down, v[i][0].w * down,
                              v[i][1].x * down, v[i][1].y * down, v[i][1].z * down, v[i][1].w * down};
          uint32_t w[4][C::kParts];
#pragma unroll
          for (int j = 0; j < 4; ++j) split<T>(f[2 * j], f[2 * j + 1], w[j]);
          // the first two parts' columns one behind the other, the third in blocks of its own
#pragma unroll
          for (int part = 0; part < C::kParts; ++part) {
            const int c = part < 2 ? part * (q.rank16 / 8) + c8 : 16 * RB + c8;
            st_shared_v4(dst + (c >> 3) * kBlockBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4), w[0][part], w[1][part], w[2][part], w[3][part]);
          }
        }
      }
      fence_async_shared();
      mbar_arrive(full(s));
      if (it + 2 < n) load();
      if (it + 4 < n) find(chunk0 + it + 4);
    }
  } else if (n > 0) {
    // ---- tensor cores ----
    bool ok = true;
    for (int it = 0; it < n; ++it) {
      const int s = it % C::kStages;
      if (!(ok = all_lanes(mbar_wait(wctx, full(s), (it / C::kStages) & 1, 0x43)))) break;
      if (!(ok = all_lanes(mbar_wait(wctx, landed(s), (it / C::kStages) & 1, 0x46)))) break;
      fence_async_shared();
      tc_fence_after_sync();
      const uint32_t a = ring + s * C::kStageBytes, b = a + C::kRows;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const uint64_t ad = umma_smem_desc_sw128(a + half * 2 * kBlockBytes + kk * 2048, kBlockBytes, 1024);
          umma_f16_elect(tmem + half * C::kHalf, ad, umma_smem_desc_sw128(b + kk * 2048, kBlockBytes, 1024), q.idesc2, it + kk > 0 ? 1u : 0u);
          if (C::kParts == 3)
            umma_f16_elect(tmem + half * C::kHalf + q.rank16, ad, umma_smem_desc_sw128(b + 2 * C::kPart + kk * 2048, kBlockBytes, 1024), q.idesc1,
                           1u);
        }
      }
      tc_commit_elect(freed(s));
    }
    if (ok) tc_commit_elect(bar_sums);
  }

  // The cluster's CTAs share the slab's columns: every CTA leaves its sums of a share in the ring of the CTA that adds them up, once
  // all rings are drained.
  const bool have = warp < C::kVecWarps && n > 0 && all_lanes(mbar_wait_long(wctx, bar_sums, 0, 0x44));
  __syncwarp();
  if (S > 1) cluster_sync();
  else __syncthreads();
  const int cols = kSlab >> q.cluster_log;   // at least 32: a warp's columns belong to one CTA
  if (warp < C::kVecWarps) {
    tc_fence_after_sync();
    const int half = warp >> 2, col = threadIdx.x & (cols - 1);
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21) + half * C::kHalf;
    const uint32_t to = cluster_map_shared(ring + (rank * q.rank16 * cols + col) * 4, threadIdx.x / cols);
    const float scale = is_a ? 1.f : __ldg(p.scales + adapter), c = scale * up;
    uint32_t redo = far ? ~0u : 0u;   // 16 ranks a bit
    const auto put = [&](int j, float sum) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + j * cols * 4), "f"(sum) : "memory"); };
    for (int b = 0; b < q.rank16 / 16; ++b) {
      float sum[16] = {};
      if (have) {
        uint32_t x[16], small[16];
        tmem_ld(lanes + b * 16, x);
        tmem_ld(lanes + q.rank16 + b * 16, small);
        tmem_wait_ld(x);
        tmem_wait_ld(small);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          sum[i] = fmaf(__uint_as_float(small[i]), 1.f / (1 << kLowUp<T>), __uint_as_float(x[i]));
          // (an infinite row or number makes NaN of the parts that it meets: zeros, or infinities of the other sign)
          if (!(fabsf(sum[i]) <= 3.4028234e38f)) redo |= 1u << b;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) put(b * 16 + i, c * sum[i]);
    }
    if (have && redo != 0u && col0 + threadIdx.x < width)
      for (int j = 0; j < p.rank; j += 4)
        if (redo >> (j >> 4) & 1u) {
          const float4 sum = plain_sums<T>(p, is_a, begin + chunk0 * 64, begin + min(count, (chunk0 + n) * 64), col0 + threadIdx.x, j);
          put(j, scale * sum.x);
          put(j + 1, scale * sum.y);
          put(j + 2, scale * sum.z);
          put(j + 3, scale * sum.w);
        }
    tc_fence_before_sync();
  }
  __syncwarp();
  if (S > 1) cluster_sync();
  else __syncthreads();
  tc_fence_after_sync();
  if (warp == C::kMmaWarp) tmem_dealloc(tmem, C::kTmemCols);
  const int64_t mine = col0 + rank * cols;
  if (S == 8) add_parts<T, 8, C::kThreads>(p, ring, q.rank16, is_a, adapter, mine);
  else if (S == 4) add_parts<T, 4, C::kThreads>(p, ring, q.rank16, is_a, adapter, mine);
  else if (S == 2) add_parts<T, 2, C::kThreads>(p, ring, q.rank16, is_a, adapter, mine);
  else add_parts<T, 1, C::kThreads>(p, ring, q.rank16, is_a, adapter, mine);
}

template <typename T, int RB>
ks_status_t launch_grad(const char* where, const GradParams& q, const CUtensorMap (&maps)[2], int64_t items, cudaStream_t stream) {
  using C = GradCfg<T, RB>;
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev >= 0 && dev < 64 && !done[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(lora_weight_grad_kernel<T, RB>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
      if (e != cudaSuccess) return cuda_status(e, where);
      done[dev] = true;
    }
  }
  launch_programmatic_cluster(lora_weight_grad_kernel<T, RB>, static_cast<unsigned>(items << q.cluster_log), 1u << q.cluster_log,
                              true, C::kThreads, C::kSmem, stream, q, maps[0], maps[1]);
  KSB_CHECK_LAUNCH(where);
  return KS_SUCCESS;
}

}  // namespace

bool lora_tile_takes(const LoraPass& p) {
  const auto rows16 = [](const void* m, int64_t ld) { return aligned16(m) && ld % 8 == 0; };
  return p.rank % 8 == 0 && p.rank <= 128 && p.d_in % 8 == 0 && p.d_out % 8 == 0 && aligned16(p.u) && aligned16(p.v) && aligned16(p.inner) &&
         rows16(p.in, p.ld_in) && rows16(p.base, p.ld_base) && rows16(p.out, p.ld_out);
}

ks_status_t lora_tile_pass(const char* where, const LoraPass& p, bool forward, ks_dtype_t dtype, cudaStream_t stream) {
  TileParams q = {};
  q.p = p;
  q.fault_word = kernel_fault_word();
  q.rank16 = (p.rank + 15) / 16 * 16;
  const uint32_t fmt = dtype == KS_DTYPE_F16 ? 0u : 1u;
  q.idesc1 = umma_instr_desc(fmt, fmt, 0u, forward ? 0u : 1u, kTile, static_cast<uint32_t>(q.rank16));
  q.idesc2 = umma_instr_desc(fmt, fmt, 0u, forward ? 0u : 1u, kTile, kChunk);
  const int64_t tiles = lora_tile_bound(p.rows, p.adapters, kTile);
  const bool wide = p.rank > 64;
  const int64_t room = static_cast<int64_t>(sm_count()) * (wide ? 1 : 2);
  // the largest cluster with which all tiles that there can be run at a time
  while ((2 << q.cluster_log) <= kMaxCluster && tiles << (q.cluster_log + 1) <= room) ++q.cluster_log;
  q.in_chunks = static_cast<int>((p.d_in + kChunk - 1) / kChunk);
  q.out_chunks = static_cast<int>((p.d_out + kChunk - 1) / kChunk);
  if (tiles << q.cluster_log > INT32_MAX) KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, std::string(where) + ": grid exceeds CUDA grid limits");
#define KSB_LORA_TILE(T, FWD)                                                      \
  (p.rank <= 32   ? launch_tile<T, 0, FWD>(where, q, tiles, stream)                \
   : p.rank <= 64 ? launch_tile<T, 1, FWD>(where, q, tiles, stream)                \
                  : launch_tile<T, 2, FWD>(where, q, tiles, stream))
  if (dtype == KS_DTYPE_F16) return forward ? KSB_LORA_TILE(__half, true) : KSB_LORA_TILE(__half, false);
  return forward ? KSB_LORA_TILE(__nv_bfloat16, true) : KSB_LORA_TILE(__nv_bfloat16, false);
#undef KSB_LORA_TILE
}

bool lora_weight_grad_takes(const LoraWeightGrad& p) {
  return p.rank % 8 == 0 && p.rank <= 128 && p.k % 8 == 0 && p.n % 8 == 0 && p.ld_x % 8 == 0 && p.ld_d_out % 8 == 0 && aligned16(p.x) &&
         aligned16(p.d_out) && aligned16(p.d_a) && aligned16(p.d_b) && aligned16(p.g) && aligned16(p.h);
}

ks_status_t lora_weight_grad_pass(const char* where, const LoraWeightGrad& p, ks_dtype_t dtype, cudaStream_t stream) {
  GradParams q = {};
  q.p = p;
  q.fault_word = kernel_fault_word();
  q.rank16 = (p.rank + 15) / 16 * 16;
  const uint32_t fmt = dtype == KS_DTYPE_F16 ? 0u : 1u;
  q.idesc2 = umma_instr_desc(fmt, fmt, 1u, 1u, 128u, static_cast<uint32_t>(2 * q.rank16));
  q.idesc1 = umma_instr_desc(fmt, fmt, 1u, 1u, 128u, static_cast<uint32_t>(q.rank16));
  q.slabs_a = static_cast<int>((p.k + kSlab - 1) / kSlab);
  q.slabs = q.slabs_a + static_cast<int>((p.n + kSlab - 1) / kSlab);
  const bool wide = p.rank > 64;
  const int64_t items = static_cast<int64_t>(p.adapters) * q.slabs;
  const int64_t room = static_cast<int64_t>(sm_count()) * (wide ? 1 : 2);
  // CTAs of a slab: as many as run at a time, and twice that where four chunks are left to each, since adapters without rows
  // leave SMs idle (16384 rows, 4 of 8 adapters, rank 64: 154 us for both launches against 194; all 8 158 / 161; 2 of 2 158 / 149)
  const auto worth = [&](int log) {
    const int64_t ctas = items << log;
    return p.rows > 32 << log && (ctas <= room || (ctas <= 2 * room && p.rows / p.adapters >= 128 << log));
  };
  while ((2 << q.cluster_log) <= kMaxCluster && worth(q.cluster_log + 1)) ++q.cluster_log;
  if (items << q.cluster_log > INT32_MAX) KSB_FAIL(KS_ERROR_UNSUPPORTED_SHAPE, std::string(where) + ": grid exceeds CUDA grid limits");
  CUtensorMap maps[2] = {};
  if (p.rows > 0) {   // (without rows nothing is copied)
    const auto encode = [&](CUtensorMap* m, const void* base, int64_t width, int64_t ld) {
      const uint64_t dims[2] = {static_cast<uint64_t>(width), static_cast<uint64_t>(p.rows)}, stride = static_cast<uint64_t>(ld) * 2;
      const uint32_t box[2] = {64, 64};
      return tma_encode(m, dtype == KS_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, &stride,
                        box, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    if (!encode(&maps[0], p.x, p.k, p.ld_x) || !encode(&maps[1], p.d_out, p.n, p.ld_d_out))
      KSB_FAIL(KS_ERROR_INTERNAL, std::string(where) + ": tensor map rejected");
  }
  if (dtype == KS_DTYPE_F16)
    return wide ? launch_grad<__half, 2>(where, q, maps, items, stream) : launch_grad<__half, 1>(where, q, maps, items, stream);
  return wide ? launch_grad<__nv_bfloat16, 2>(where, q, maps, items, stream) : launch_grad<__nv_bfloat16, 1>(where, q, maps, items, stream);
}

}  // namespace sm100
}  // namespace ksb
