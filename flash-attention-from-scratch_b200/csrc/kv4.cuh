// The 4-bit cache row, shared by the kernels that write, read back and attend
// over it.
//
// One row holds K (or V) of one token of one kv head: head_dim values in groups
// of 32, each group with an fp16 scale and an fp16 low,
//     value = low + scale * code,   code in 0..15.
// NG = head_dim / 32 groups. Bytes of a row (80 at head_dim 128, 40 at 64):
//     [0, D / 2)              codes
//     [D / 2, D / 2 + 2 NG)   scales
//     [.., + 2 NG)            lows
// The codes stand in the order in which the decode kernel's tensor-core
// fragments take them, so that it unpacks with masks alone:
//     K: 32-bit word t * NG + w holds dims 32 w + 8 t + e at bits 4 e  (e < 8)
//     V: 16-bit word g * NG + w holds columns 32 w + 4 g + j at bits 4 j (j < 4)
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace fab {

// n / d for n < 2^31 by a product: with 2^s >= d > 2^(s - 1), s >= 1, the factor
// m = ceil(2^(31 + s) / d) is below 2^32, and m d - 2^(31 + s) < 2^s makes
// n m >> (31 + s) exact. d = 1: factor 0 stands for it.
struct FastDiv {
  uint32_t factor, shift;
  FastDiv() = default;
  explicit FastDiv(int64_t d) {
    shift = 1;
    while ((int64_t(1) << shift) < d) ++shift;
    factor = d == 1 ? 0u
                    : static_cast<uint32_t>(((uint64_t(1) << (31 + shift)) + d - 1) /
                                            static_cast<uint64_t>(d));
    --shift;
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
    return factor == 0u ? n : __umulhi(n, factor) >> shift;
  }
};

// `total` stages dealt out in equal runs to n workers (one per stage, if that is
// fewer): the first `more` workers have size + 1 stages, the others `size`.
struct Runs {
  unsigned int workers, size, more;
  __device__ __forceinline__ Runs(unsigned int total, unsigned int n) {
    workers = min(n, total);
    size = workers == 0 ? 0 : total / workers;
    more = total - size * workers;
  }
  // First stage of worker i.
  __device__ __forceinline__ unsigned int begin(unsigned int i) const {
    return size * i + min(i, more);
  }
  // The worker that has stage s.
  __device__ __forceinline__ unsigned int of(unsigned int s) const {
    const unsigned int big = more * (size + 1);
    return s < big ? s / (size + 1) : more + (s - big) / size;
  }
};

template <int D>
struct Kv4Row {
  static constexpr int NG = D / 32;
  static constexpr int CODES = D / 2;
  static constexpr int BYTES = D / 2 + 4 * NG;
};

__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  return pack_half2(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

}  // namespace fab
