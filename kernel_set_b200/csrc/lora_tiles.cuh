// Device code shared by the adapters' tensor-core kernels: 16-bit pairs, the scale of an inner vector, and where a tile lies.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "lora_math.cuh"

namespace ksb {
namespace sm100 {

template <typename T>
struct Pair;   // two 16-bit numbers in a word
template <>
struct Pair<__half> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
};
template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
};

// An inner vector is a sum in fp32; it enters the next product as a sum of 16-bit numbers, the first the nearest to it, each further one
// the nearest to what is left: three of bf16 hold all 24 bits, two of f16 hold 22. (Two of bf16, 2^-18 of the number, changed one in
// 400 of the outputs in their last place.) f16 has few exponents: the vector is scaled (row_scale) so that its largest number is
// just below 2^15, and the second part is kept 2^kLowUp times as large, its sums brought back behind the product. A number is
// then held to 2^-22 of itself down to 2^-28 of the largest, and to 2^-50 of the largest below.
template <typename T>
constexpr int kInnerParts = std::is_same<T, __half>::value ? 2 : 3;
template <typename T>
constexpr int kLowUp = std::is_same<T, __half>::value ? 11 : 0;
template <typename T>
constexpr int kTop = std::is_same<T, __half>::value ? 14 : 0;   // exponent of the largest number of a scaled vector

template <typename T>
__device__ __forceinline__ void split(float f0, float f1, uint32_t (&part)[kInnerParts<T>]) {
#pragma unroll
  for (int i = 0; i < kInnerParts<T>; ++i) {
    part[i] = Pair<T>::pack(f0, f1);
    const float2 w = Pair<T>::unpack(part[i]);
    f0 = (f0 - w.x) * static_cast<float>(1 << kLowUp<T>);
    f1 = (f1 - w.y) * static_cast<float>(1 << kLowUp<T>);
  }
}

// The power of two 2^-e for a vector whose largest magnitude is `most`, so that most 2^-e is in [2^kTop, 2^(kTop+1)) where possible, and 2^e.
// It keeps what f16 could not hold (sums beyond 65504, small ones whose low part would vanish); 1 for zeros and non-finite vectors.
template <typename T>
__device__ __forceinline__ void row_scale(float most, float* down, float* up) {
  uint32_t e = (__float_as_uint(most) >> 23) & 255u;
  if (e == 0u || e == 255u) e = 127u + kTop<T>;
  e = e > 253u + kTop<T> ? 253u + kTop<T> : e;
  e = e < kTop<T> + 1u ? kTop<T> + 1u : e;
  *down = __uint_as_float((254u + kTop<T> - e) << 23);
  *up = __uint_as_float((e - kTop<T>) << 23);
}

// How far the numbers of an adapter's vectors lie apart: beyond 2^33 the smallest would be off by more than 2^-17 of themselves.
__device__ __forceinline__ bool far_apart(float most, float least) { return !(most <= 3.4028234e38f) || least < most * 1.1641532e-10f; }

// Where tile `index` lies: adapter (`adapters` for the rows without one, -1 past the last tile), first place and row count.
struct TilePlace {
  int adapter;
  int count;
  int64_t place;
};

// Found by one warp: a lane counts the tiles of a run of adapters, the one whose run holds the tile walks it again.
template <int TILE>
__device__ __forceinline__ TilePlace find_tile(const int32_t* __restrict__ offsets, int adapters, int64_t rows, int64_t index) {
  const int lane = threadIdx.x & 31;
  const int groups = adapters + 1;
  const int run = (groups + 31) / 32;
  const int first = lane * run < groups ? lane * run : groups;
  const int last = first + run < groups ? first + run : groups;
  const auto begin_of = [&](int g) { return g > adapters ? rows : lora_offset(offsets, g, rows); };
  int64_t mine = 0;
#pragma unroll 4
  for (int g = first; g < last; ++g) {
    const int64_t n = begin_of(g + 1) - begin_of(g);
    mine += n > 0 ? (n + TILE - 1) / TILE : 0;
  }
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += t;
  }
  TilePlace f{-1, 0, 0};
  const bool here = index < upto && index >= upto - mine;
  if (here) {
    int64_t left = index - (upto - mine);
    for (int g = first; g < last; ++g) {
      const int64_t b = begin_of(g), n = begin_of(g + 1) - b;
      const int64_t tiles = n > 0 ? (n + TILE - 1) / TILE : 0;
      if (left < tiles) {
        f.adapter = g;
        f.place = b + left * TILE;
        const int64_t rest = n - left * TILE;
        f.count = static_cast<int>(rest < TILE ? rest : TILE);
        break;
      }
      left -= tiles;
    }
  }
  const unsigned who = __ballot_sync(0xffffffffu, here);
  if (who == 0u) return f;
  const int src = __ffs(who) - 1;
  f.adapter = __shfl_sync(0xffffffffu, f.adapter, src);
  f.count = __shfl_sync(0xffffffffu, f.count, src);
  f.place = __shfl_sync(0xffffffffu, f.place, src);
  return f;
}

}  // namespace sm100
}  // namespace ksb
