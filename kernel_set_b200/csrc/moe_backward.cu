// Gradients of a routed layer's steps: the gate's (softmax, top-k, weights optionally renormalised), the row
// gather's and the weighted sum's. No counterpart in the reference's C ABI.
//
// All three are bound by memory: a row is read and written once, sums are held in fp32 and rounded once, and every
// sum has one order (slots in turn; threads of a CTA by a fixed tree), so results repeat to the bit.
#include <mutex>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "kernel_set/ext/moe_backward.h"
#include "lora_tiles.cuh"
#include "moe_rows.cuh"
#include "sm100_host.cuh"
#include "sm100_ptx.cuh"

namespace ksb {
namespace {

// 16 bytes of a row, or one element. They stay packed until they are used (as an array of 16-bit elements each takes a register of
// its own: 126 a thread against 72 where eight pieces are in flight).
template <typename T, int VEC>
struct Piece {
  static_assert(VEC * sizeof(T) == 16, "");
  uint4 w;
  __device__ __forceinline__ static Piece load(const T* p) { return {*reinterpret_cast<const uint4*>(p)}; }
  __device__ __forceinline__ static Piece stream(const T* p) { return {__ldcs(reinterpret_cast<const uint4*>(p))}; }   // read once
  __device__ __forceinline__ void unpack(float (&f)[VEC]) const {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (VEC == 4) {
        f[i] = __uint_as_float(x[i]);
      } else {
        const float2 v = sm100::Pair<T>::unpack(x[i]);
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
      }
    }
  }
  __device__ __forceinline__ static void store(T* p, const float (&f)[VEC]) {
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (VEC == 4) x[i] = __float_as_uint(f[i]);
      else x[i] = sm100::Pair<T>::pack(f[2 * i], f[2 * i + 1]);
    }
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(x[0], x[1], x[2], x[3]));
  }
};
template <typename T>
struct Piece<T, 1> {
  T v;
  __device__ __forceinline__ static Piece load(const T* p) { return {*p}; }
  __device__ __forceinline__ static Piece stream(const T* p) { return {*p}; }
  __device__ __forceinline__ void unpack(float (&f)[1]) const { f[0] = to_f32<T>(v); }
  __device__ __forceinline__ static void store(T* p, const float (&f)[1]) { *p = from_f32<T>(f[0]); }
};

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
    const float zero[VEC] = {};
    for (int64_t c = threadIdx.x; c < pieces; c += kRowThreads) Piece<T, VEC>::store(dp + c * VEC, zero);
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
        pv[u] = Piece<T, VEC>::stream(p + c * VEC);
        gv[u] = Piece<T, VEC>::load(g + c * VEC);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t c = c0 + u * kRowThreads;
      if (c >= pieces) continue;
      float d[VEC], x[VEC];
      gv[u].unpack(d);
      pv[u].unpack(x);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        dot = fmaf(d[i], x[i], dot);
        d[i] *= w;
      }
      Piece<T, VEC>::store(dp + c * VEC, d);
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
// Up to kScanPairs pairs a CTA looks through all ids itself for its token's rows, from L2, without a second launch, unless the
// CTAs together read more than kScanIds ids: 128 tokens x 8 rows of 7168 bf16 3.6 us against 6.4 with the map, 256 tokens 7.0 / 9.1,
// 512 tokens 17.4 / 13.8, 4096 tokens x 1 row of 4096 61.8 / 16.0. Beyond that the rows come from the inverse map, looked up again as ks_moe_unpermute does. These are two dependent reads in front of the rows':
// the warps stay and go from item to item (a part of a token), and ask for the next item's rows before they read this one's. Up to 8
// rows a token in whole 16-byte pieces come by bulk copies, two items ahead in shared memory (permute_backward_bulk_kernel);
// otherwise into registers, 8 pieces a lane. 4096 tokens x 8 rows of 7168 bf16, an eighth of them dropped (470 MB, 72 us at the rate of a
// copy): 96 us; a CTA per 2 KB of a token with the three reads one behind the other 176.
constexpr int kScanPairs = 4096;
constexpr int64_t kScanIds = 1 << 22;
constexpr int kMapCtasPerSm = 4;   // (more of them in flight are slower: 114 us against 157 with 6)

// One warp: piece c of `token`, whose rows are `mine` (lane k: slot k) and look_up(k) for the slots from 32 on.
template <typename T, int VEC, typename LookUp>
__device__ __forceinline__ void add_rows(T* __restrict__ d_input, const T* __restrict__ d_permuted, int64_t token, int64_t c, int64_t pieces,
                                         int64_t hidden, int top_k, int32_t mine, const LookUp& look_up) {
  constexpr int kAtOnce = 8;
  float acc[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
  for (int k0 = 0; k0 < top_k; k0 += kAtOnce) {
    if (k0 > 0 && k0 % 32 == 0) mine = look_up(k0 + (threadIdx.x & 31));
    Piece<T, VEC> v[kAtOnce];
    bool take[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int32_t row = __shfl_sync(0xffffffffu, mine, (k0 + j) & 31);   // (-1 from top_k on)
      take[j] = row >= 0;
      if (take[j] && c < pieces) v[j] = Piece<T, VEC>::stream(d_permuted + static_cast<int64_t>(row) * hidden + c * VEC);
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (!take[j] || c >= pieces) continue;
      float x[VEC];
      v[j].unpack(x);
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += x[i];
    }
  }
  if (c < pieces) Piece<T, VEC>::store(d_input + token * hidden + c * VEC, acc);
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kRowThreads)
permute_backward_scan_kernel(T* __restrict__ d_input, const T* __restrict__ d_permuted, const int32_t* __restrict__ ids, int64_t pairs,
                             int top_k, int64_t hidden, unsigned chunks) {
  extern __shared__ int32_t rows[];   // of the token's slots
  sm100::grid_dependency_wait();
  const int64_t token = blockIdx.x / chunks;
  const int64_t chunk = blockIdx.x - token * chunks;
  const int64_t first = token * top_k;
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
  __syncthreads();
  const auto look_up = [&](int k) -> int32_t { return k < top_k ? rows[k] : -1; };
  add_rows<T, VEC>(d_input, d_permuted, token, chunk * kRowThreads + threadIdx.x, hidden / VEC, hidden, top_k,
                   look_up(threadIdx.x & 31), look_up);
}

// `chunks` items of 32 pieces per token; warp w of `stride` takes the items w, w + stride, ... (token_step * chunks +
// chunk_step = stride).
template <typename T, int VEC>
__global__ void __launch_bounds__(kRowThreads)
permute_backward_kernel(T* __restrict__ d_input, const T* __restrict__ d_permuted, const int32_t* __restrict__ ids,
                        const int32_t* __restrict__ inverse, int64_t tokens, int top_k, int64_t hidden, int64_t chunks, int64_t token_step,
                        int64_t chunk_step) {
  sm100::grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t pieces = hidden / VEC, pairs = tokens * top_k;
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * (kRowThreads / 32) + (threadIdx.x >> 5);
  int64_t token = warp / chunks, chunk = warp - token * chunks;
  const auto row_of = [&](int64_t t, int k) -> int32_t {   // the row of a token's slot
    return t < tokens && k < top_k ? check_row(__ldg(inverse + t * top_k + k), ids, t * top_k + k, pairs) : -1;
  };
  int32_t mine = row_of(token, lane);
  while (token < tokens) {
    int64_t next = token + token_step, next_chunk = chunk + chunk_step;
    if (next_chunk >= chunks) {
      next_chunk -= chunks;
      ++next;
    }
    const int32_t after = row_of(next, lane);
    add_rows<T, VEC>(d_input, d_permuted, token, chunk * 32 + lane, pieces, hidden, top_k, mine,
                     [&](int k) { return row_of(token, k); });
    mine = after;
    token = next;
    chunk = next_chunk;
  }
}

// The same for up to kBulkSlots rows a token, 16 bytes at a time throughout: a warp has three buffers and brings the rows' segments
// of `seg` bytes into them by bulk copies, two items ahead of the one that it adds up. 16 warps of an SM are needed to add
// up what arrives: 8 with twice the buffers 107 us, 4 with four times 133.
constexpr int kBulkSlots = 8;
constexpr int kBulkWarps = 4;
constexpr int kBulkBuffers = 3;    // (what asks two items ahead and reads one)
constexpr int kBulkBytes = 4096;   // of a buffer
constexpr int kBulkCtasPerSm = 4;
constexpr int kBulkSmem = kBulkWarps * kBulkBuffers * (kBulkBytes + 8) + 16;
static_assert(kBulkCtasPerSm * (kBulkSmem + 1024) <= 233472, "shared memory");

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
               "r"(bar)
               : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kBulkWarps * 32)
permute_backward_bulk_kernel(T* __restrict__ d_input, const T* __restrict__ d_permuted, const int32_t* __restrict__ ids,
                             const int32_t* __restrict__ inverse, int64_t tokens, int top_k, int64_t hidden, int64_t chunks, int seg,
                             int64_t token_step, int64_t chunk_step, unsigned int* fault_word) {
  constexpr int kVec = 16 / sizeof(T);
  extern __shared__ __align__(128) unsigned char bulk_smem[];
  const int w = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t buffers = sm100::smem_u32(bulk_smem) + w * kBulkBuffers * kBulkBytes;
  const uint32_t all_bars = sm100::smem_u32(bulk_smem) + kBulkWarps * kBulkBuffers * kBulkBytes;
  const uint32_t bars = all_bars + w * kBulkBuffers * 8;
  const sm100::WaitCtx wctx{all_bars + kBulkWarps * kBulkBuffers * 8, fault_word};
  if (threadIdx.x == 0) {
    for (int i = 0; i < kBulkWarps * kBulkBuffers; ++i) sm100::mbar_init(all_bars + 8 * i, 1);
    *reinterpret_cast<uint32_t*>(bulk_smem + (wctx.abort_at - sm100::smem_u32(bulk_smem))) = 0u;
    sm100::fence_barrier_init();
  }
  __syncthreads();
  sm100::grid_dependency_wait();
  const int64_t row_bytes = hidden * static_cast<int64_t>(sizeof(T)), pairs = tokens * top_k;
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * kBulkWarps + w;
  struct Item {
    int64_t token, chunk;
  };
  const auto after = [&](Item i) {
    i.token += token_step;
    i.chunk += chunk_step;
    if (i.chunk >= chunks) {
      i.chunk -= chunks;
      ++i.token;
    }
    return i;
  };
  const auto row_of = [&](const Item& i) -> int32_t {   // lane k: the row of the token's slot k
    const int64_t pair = i.token * top_k + lane;
    return i.token < tokens && lane < top_k ? check_row(__ldg(inverse + pair), ids, pair, pairs) : -1;
  };
  const auto bytes_of = [&](const Item& i) { return static_cast<uint32_t>(min(static_cast<int64_t>(seg), row_bytes - i.chunk * seg)); };
  uint32_t live[kBulkBuffers] = {}, parity = 0u;   // slots in each buffer
  const auto ask = [&](const Item& i, int32_t row, int b) {
    const uint32_t mask = __ballot_sync(0xffffffffu, row >= 0);
    if (mask != 0u) {
      const uint32_t bytes = bytes_of(i);
      if (lane == 0) sm100::mbar_arrive_expect_tx(bars + 8 * b, bytes * __popc(mask));
      __syncwarp();
      if (row >= 0)
        bulk_load(buffers + b * kBulkBytes + lane * seg, reinterpret_cast<const char*>(d_permuted) + row * row_bytes + i.chunk * seg, bytes,
                  bars + 8 * b);
    }
    return mask;
  };
  Item now = {warp / chunks, warp % chunks};
  Item ahead = after(now);
  live[0] = ask(now, row_of(now), 0);
  live[1] = ask(ahead, row_of(ahead), 1);
  ahead = after(ahead);
  int32_t row = row_of(ahead);
  bool ok = true;
  while (ok && now.token < tokens) {
#pragma unroll
    for (int b = 0; b < kBulkBuffers; ++b) {
      if (!ok || now.token >= tokens) break;
      constexpr int kLast = kBulkBuffers - 1;
      live[(b + kLast) % kBulkBuffers] = ask(ahead, row, (b + kLast) % kBulkBuffers);
      ahead = after(ahead);
      row = row_of(ahead);
      const uint32_t mask = live[b];
      if (mask != 0u) {
        ok = sm100::all_lanes(sm100::mbar_wait(wctx, bars + 8 * b, parity >> b & 1u, 0x51));
        if (!ok) break;
        parity ^= 1u << b;
      }
      const uint32_t bytes = bytes_of(now), from = buffers + b * kBulkBytes;
      T* to = d_input + now.token * hidden + now.chunk * (seg / static_cast<int>(sizeof(T)));
      for (uint32_t at = lane * 16; at < bytes; at += 512) {
        Piece<T, kVec> v[kBulkSlots];
#pragma unroll
        for (int k = 0; k < kBulkSlots; ++k) v[k] = {sm100::ld_shared_v4(from + (k < top_k ? k * seg : 0) + at)};
        float acc[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) acc[i] = 0.f;
#pragma unroll
        for (int k = 0; k < kBulkSlots; ++k) {
          if (!(mask >> k & 1u)) continue;
          float x[kVec];
          v[k].unpack(x);
#pragma unroll
          for (int i = 0; i < kVec; ++i) acc[i] += x[i];
        }
        Piece<T, kVec>::store(to + at / sizeof(T), acc);
      }
      live[b] = 0u;
      __syncwarp();   // (the buffer is read: the next item's copies may overwrite it)
      now = after(now);
    }
  }
#pragma unroll
  for (int b = 0; b < kBulkBuffers; ++b)   // after a wait that ran out: the warp's own copies
    if (!ok && live[b] != 0u) sm100::mbar_wait(wctx, bars + 8 * b, parity >> b & 1u, 0x52);
}

// ---------------------------------------------------------------------------------
// gate
// ---------------------------------------------------------------------------------
// A warp per token; a lane holds the logits of VEC neighbouring experts at a time in registers, COUNT times. Without
// renormalisation d = -p s for all experts, otherwise zeros; then the lane of a chosen slot writes that expert's number once more,
// with the slots of the expert added in turn (behind the row's stores, in the same warp). Bound by memory, once read and
// once written: 16384 tokens x 256 experts in bf16 take 14 us cold. (Every lane comparing its experts with all slots, two bytes a load: 23.5 us cold.)
template <typename T, int VEC>
__device__ __forceinline__ void load_gate(const T* p, float (&v)[VEC]) {
  if constexpr (VEC * sizeof(T) == 2 || (VEC == 1)) v[0] = to_f32<T>(*p);
  else {
    using Word = std::conditional_t<VEC * sizeof(T) == 16, uint4, std::conditional_t<VEC * sizeof(T) == 8, uint2, uint32_t>>;
    const Word w = *reinterpret_cast<const Word*>(p);
    const T* t = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32<T>(t[i]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_gate(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) *p = from_f32<T>(v[0]);
  else {
    using Word = std::conditional_t<VEC * sizeof(T) == 16, uint4, std::conditional_t<VEC * sizeof(T) == 8, uint2, uint32_t>>;
    Word w;
    T* t = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = from_f32<T>(v[i]);
    *reinterpret_cast<Word*>(p) = w;
  }
}

constexpr int kGateThreads = 256;

template <typename T, int VEC, int COUNT>
__global__ void __launch_bounds__(kGateThreads)
gate_backward_kernel(T* d_logits, const float* __restrict__ d_weights, const float* __restrict__ weights,
                     const int32_t* __restrict__ indices, const T* logits, int64_t tokens, int experts, int top_k,
                     int renormalize) {
  sm100::grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * (kGateThreads / 32) + (threadIdx.x >> 5);
  if (token >= tokens) return;   // whole warp
  const T* row = logits + token * experts;
  float v[COUNT][VEC];
  if (!renormalize) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      const int e = (i * 32 + lane) * VEC;
      if (e < experts) load_gate<T, VEC>(row + e, v[i]);
    }
  }
  int idx = -1;
  float w = 0.f, dw = 0.f, own = 0.f;
  if (lane < top_k) {
    idx = __ldg(indices + token * top_k + lane);
    w = __ldg(weights + token * top_k + lane);
    dw = __ldg(d_weights + token * top_k + lane);
    if (idx < 0 || idx >= experts) {
      idx = -1;
      w = dw = 0.f;
    } else if (!renormalize) {
      own = to_f32<T>(row[idx]);
    }
  }
  float s = w * dw;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const float add = renormalize ? w * (dw - s) : w * dw;
  float mine = 0.f;   // the slot's expert's number
  if (!renormalize) {
    float mx = -__int_as_float(0x7f800000), sum = 0.f;
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
      if ((i * 32 + lane) * VEC < experts) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) mx = fmaxf(mx, v[i][j]);
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
      if ((i * 32 + lane) * VEC < experts) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum += v[i][j] = expf(v[i][j] - mx);
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float scale = -s / sum;
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] *= scale;
    mine = expf(own - mx) * scale;
  } else {
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = 0.f;
  }
  for (int k = 0; k < top_k; ++k) {
    const int ek = __shfl_sync(0xffffffffu, idx, k);
    const float ak = __shfl_sync(0xffffffffu, add, k);
    if (ek == idx) mine += ak;   // (in turn, so all slots of an expert hold the same number)
  }
  T* out = d_logits + token * experts;
  __syncwarp();   // (in place: a lane overwrites logits that another has read; shuffles promise no order of memory accesses)
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    const int e = (i * 32 + lane) * VEC;
    if (e < experts) store_gate<T, VEC>(out + e, v[i]);
  }
  __syncwarp();
  if (idx >= 0) out[idx] = from_f32<T>(mine);
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
  T* o = static_cast<T*>(d_input);
  const T* x = static_cast<const T*>(d_permuted);
  const int64_t scan_chunks = (pieces + kRowThreads - 1) / kRowThreads;
  if (pairs <= kScanPairs && scan_chunks <= kScanIds / (tokens * pairs)) {
    const auto kernel = vec ? permute_backward_scan_kernel<T, kVec> : permute_backward_scan_kernel<T, 1>;
    sm100::launch_programmatic(kernel, static_cast<unsigned>(tokens * scan_chunks), kRowThreads, static_cast<size_t>(top_k) * sizeof(int32_t), s,
                               o, x, ids, pairs, top_k, hidden, static_cast<unsigned>(scan_chunks));
    KSB_CHECK_LAUNCH(where);
    return KS_SUCCESS;
  }
  sm100::StreamScratch scratch(s);   // (until both kernels are enqueued)
  int32_t* inverse = static_cast<int32_t*>(scratch.get(static_cast<size_t>(pairs) * sizeof(int32_t), kInverseScratch));
  if (inverse == nullptr) KSB_FAIL(KS_ERROR_OUT_OF_MEMORY, "ks_moe_permute_backward: workspace allocation failed");
  enqueue_inverse_permutation(inverse, ids, pairs, s);
  if (vec && top_k <= kBulkSlots) {
    static std::mutex mu;
    static bool done[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    {
      std::lock_guard<std::mutex> lock(mu);
      if (dev >= 0 && dev < 64 && !done[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(permute_backward_bulk_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBulkSmem);
        if (e != cudaSuccess) return cuda_status(e, where);
        done[dev] = true;
      }
    }
    // segments of about equal size that fit a buffer, multiples of a warp's 512 bytes
    const int64_t row_bytes = hidden * static_cast<int64_t>(sizeof(T)), most = kBulkBytes / top_k / 512 * 512;
    const int64_t chunks = (row_bytes + most - 1) / most;
    const int64_t seg = ((row_bytes + chunks - 1) / chunks + 511) / 512 * 512;
    const int64_t ctas_most = static_cast<int64_t>(sm_count()) * kBulkCtasPerSm, ctas_want = (tokens * chunks + kBulkWarps - 1) / kBulkWarps;
    const int64_t ctas = ctas_want < ctas_most ? ctas_want : ctas_most;
    sm100::launch_programmatic(permute_backward_bulk_kernel<T>, static_cast<unsigned>(ctas), kBulkWarps * 32, kBulkSmem, s, o, x, ids, inverse,
                               tokens, top_k, hidden, chunks, static_cast<int>(seg), ctas * kBulkWarps / chunks, ctas * kBulkWarps % chunks,
                               kernel_fault_word());
    KSB_CHECK_LAUNCH(where);
    return KS_SUCCESS;
  }
  const int64_t chunks = (pieces + 31) / 32;
  const int64_t items = chunks > INT64_MAX / tokens ? INT64_MAX : chunks * tokens;
  constexpr int64_t kWarps = kRowThreads / 32;
  const int64_t most = static_cast<int64_t>(sm_count()) * kMapCtasPerSm;
  const int64_t ctas = items / kWarps + 1 < most ? items / kWarps + 1 : most;
  const auto kernel = vec ? permute_backward_kernel<T, kVec> : permute_backward_kernel<T, 1>;
  sm100::launch_programmatic(kernel, static_cast<unsigned>(ctas), kRowThreads, 0, s, o, x, ids, inverse, tokens, top_k, hidden, chunks,
                             ctas * kWarps / chunks, ctas * kWarps % chunks);
  KSB_CHECK_LAUNCH(where);
  return KS_SUCCESS;
}

template <typename T>
void gate_backward(void* d_logits, const float* d_weights, const float* weights, const int32_t* indices, const void* logits, int64_t tokens,
                   int experts, int top_k, int renormalize, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>((tokens + kGateThreads / 32 - 1) / (kGateThreads / 32));
  const auto launch = [&](auto kernel) {
    sm100::launch_programmatic(kernel, grid, kGateThreads, 0, s, static_cast<T*>(d_logits), d_weights, weights, indices,
                               static_cast<const T*>(logits), tokens, experts, top_k, renormalize);
  };
  // the widest access that rows and addresses allow and that leaves no lane idle
  constexpr int kMost = 16 / sizeof(T);
  const auto fits = [&](int vec) {
    return experts % vec == 0 && experts >= 32 * vec && reinterpret_cast<uintptr_t>(d_logits) % (vec * sizeof(T)) == 0 &&
           reinterpret_cast<uintptr_t>(logits) % (vec * sizeof(T)) == 0;
  };
  const auto of = [&](auto vec) {   // up to two accesses a lane, or as many as the most experts need
    constexpr int kVec = decltype(vec)::value;
    if (experts <= 64 * kVec) launch(gate_backward_kernel<T, kVec, 2>);
    else launch(gate_backward_kernel<T, kVec, kMaxExperts / (32 * kVec)>);
  };
  if (kMost == 8 && fits(8)) of(std::integral_constant<int, kMost>());
  else if (fits(4)) of(std::integral_constant<int, 4>());
  else if (fits(2)) of(std::integral_constant<int, 2>());
  else of(std::integral_constant<int, 1>());
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
  st = poll_kernel_fault(where);
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
  const auto run = dtype == KS_DTYPE_F32 ? gate_backward<float> : dtype == KS_DTYPE_F16 ? gate_backward<__half> : gate_backward<__nv_bfloat16>;
  run(d_logits, d_weights, weights, indices, logits, num_tokens, num_experts, top_k, renormalize, s);
  KSB_CHECK_LAUNCH(where);
  return KS_SUCCESS;
}

}  // extern "C"
