// The 4-bit paged cache: quantising new tokens into their slots, and reading
// slots back (the row's layout: kv4.cuh).
//
// Quantisation of one group of 32 values x:
//     low   = fp16(min x)
//     scale = fp16((max x - low) / 15)        the quotient rounded to fp32 first
//     code  = (x - low) / scale, rounded to the nearest whole number, ties to
//             even, clamped to 0..15; 0 where the scale is 0.
// A group with a value outside fp16's finite range (only bf16 inputs have other
// finite ones) reads back as NaN: scale = low = NaN, codes 0.
#include <type_traits>

#include "kv4.cuh"
#include "launch.h"

namespace fab {
namespace {

enum : unsigned int { kSiteAppendSlot = 211, kSiteReadSlot = 212 };

struct Kv4CopyParams {
  const void* src[2];         // K and V: values (append) or rows (read)
  void* dst[2];
  long long token_stride[2];  // of the values, in elements
  long long head_stride[2];
  const long long* slots;     // [tokens]: page * bs + offset; below 0: no token
  float* weights;             // [num_blocks, hkv, bs] or null: set to 0 in the written slots
  DeviceStatus* status;
  long long num_slots;        // num_blocks * bs
  unsigned int rows;          // tokens * hkv, below 2^31
  int hkv, bs;
  FastDiv by_hkv, by_bs;
  int narrow;                 // the cache has fewer than 2^31 rows
};

// Number of the cache row of (slot, head).
__device__ __forceinline__ long long cache_row(const Kv4CopyParams& p, long long slot, int head) {
  if (p.narrow) {
    const unsigned int s = static_cast<unsigned int>(slot), page = p.by_bs.quotient(s);
    return (page * p.hkv + head) * p.bs + (s - page * p.bs);
  }
  const long long page = slot / p.bs;
  return (page * p.hkv + head) * p.bs + (slot - page * p.bs);
}

__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b, __half) {
  const __half2 r = __hmin2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b, __nv_bfloat16) {
  const __nv_bfloat162 r = __hmin2_nan(*reinterpret_cast<__nv_bfloat162*>(&a),
                                       *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b, __half) {
  const __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b, __nv_bfloat16) {
  const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a),
                                       *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float approx_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void unpack2(uint32_t v, float& lo, float& hi, __half) {
  const float2 f = __half22float2(*reinterpret_cast<__half2*>(&v));
  lo = f.x;
  hi = f.y;
}
__device__ __forceinline__ void unpack2(uint32_t v, float& lo, float& hi, __nv_bfloat16) {
  lo = __uint_as_float(v << 16);
  hi = __uint_as_float(v & 0xFFFF0000u);
}

// The 32-bit word of a row that lane (w, t) stores: of K its own 8 codes, of V half
// 2 t (of an even w) or 2 t + 1 of the groups w & ~1 and w | 1.
template <int D, bool V>
__device__ __forceinline__ int word_of(int w, int t) {
  constexpr int NG = Kv4Row<D>::NG;
  return V ? ((2 * t + (w & 1)) * NG + (w & ~1)) / 2 : t * NG + w;
}

// Four lanes per group, each with 8 of its 32 values in one 16-byte load: lane
// t of the group makes exactly the row's 32-bit K word (t, w); of V it makes the
// 16-bit words g = 2 t and 2 t + 1 of group w, and trades one of them with the
// lane of group w ^ 1, so that every lane stores one 32-bit word and a row's
// codes are one contiguous store of the warp.
template <int D, typename T, bool V>
__device__ __forceinline__ void append_row(uint8_t* dst, uint4 raw, bool real, int w, int t) {
  using R = Kv4Row<D>;
  // min and -max (the sign flipped) of the group, together in one register.
  uint32_t lo2 = min2_nan(min2_nan(raw.x, raw.y, T()), min2_nan(raw.z, raw.w, T()), T());
  uint32_t hi2 =
      max2_nan(max2_nan(raw.x, raw.y, T()), max2_nan(raw.z, raw.w, T()), T()) ^ 0x80008000u;
  uint32_t ends = min2_nan(__byte_perm(lo2, hi2, 0x5410), __byte_perm(lo2, hi2, 0x7632), T());
  ends = min2_nan(ends, __shfl_xor_sync(0xffffffffu, ends, 1), T());
  ends = min2_nan(ends, __shfl_xor_sync(0xffffffffu, ends, 2), T());
  float lo, neg_hi;
  unpack2(ends, lo, neg_hi, T());
  __half lo_h = __float2half_rn(lo);
  const float low = __half2float(lo_h);
  // The range over 15, correctly rounded: with y = RN(1 / 15) and q = RN(range y), the
  // residual range - 15 q is exact in an fma and RN(q + residual y) is the quotient
  // (P. Markstein, IBM Journal of Research and Development 34, 1990).
  const float range = -neg_hi - low;
  constexpr float kFifteenth = 1.f / 15.f;
  const float about = range * kFifteenth;
  __half scale_h =
      __float2half_rn(fmaf(fmaf(-15.f, about, range), kFifteenth, about));
  if (!(fabsf(lo) <= 65504.f && fabsf(neg_hi) <= 65504.f))
    lo_h = scale_h = __ushort_as_half(0x7fff);  // NaN
  const float scale = __half2float(scale_h);
  const bool live = scale > 0.f;  // not 0, not NaN
  const float inv = live ? approx_rcp(scale) : 0.f;
  float x[8];
  unpack2(raw.x, x[0], x[1], T());
  unpack2(raw.y, x[2], x[3], T());
  unpack2(raw.z, x[4], x[5], T());
  unpack2(raw.w, x[6], x[7], T());
  // Codes by adding 1.5 2^23, which rounds the quotient to a whole number in the
  // sum's low bits; the sums' other bits add up to a constant.
  constexpr float kBig = 12582912.f;
  constexpr uint32_t kBits = 0x4B400000u;
  constexpr uint32_t kAll = kBits * 0x11111111u;  // kBits << 0, 4, ..., 28
  const uint64_t low2 = f2_pack(-low, -low), inv2 = f2_pack(inv, inv);
  const uint64_t big2 = f2_pack(kBig, kBig), unbig2 = f2_pack(-kBig, -kBig);
  const uint64_t minus2 = f2_pack(-1.f, -1.f);
  float d[8], off = 0.f;
  uint32_t sum = 0;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint64_t r = f2_mul(f2_add(f2_pack(x[i], x[i + 1]), low2), inv2);
    const uint64_t n = f2_add(r, big2);
    float n0, n1;
    f2_unpack(f2_fma(f2_add(n, unbig2), minus2, r), d[i], d[i + 1]);
    f2_unpack(n, n0, n1);
    sum += __float_as_uint(n0) * (1u << (4 * i));
    sum += __float_as_uint(n1) * (1u << (4 * i + 4));
    off = fmaxf(off, fmaxf(fabsf(d[i]), fabsf(d[i + 1])));
  }
  uint32_t word = live ? sum - kAll : 0u;
  // The quotient above is off by a few fp32 roundings (below 2^-17 of a code). Next
  // to a half it is the sign of x - low - (n + 1/2) scale that decides, exact in 64
  // bits, and of an exact half the even code stands. A scale below fp16's normal
  // range is rounded so coarsely that quotients can pass 15.5.
  if (live && (off > 0.5f - 0x1p-16f || scale < 0x1p-14f)) {
    if (scale < 0x1p-14f) {
      word = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double q = (static_cast<double>(x[i]) - low) / static_cast<double>(scale);
        word |= static_cast<uint32_t>(fmin(fmax(rint(q), 0.0), 15.0)) << (4 * i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (fabsf(d[i]) <= 0.5f - 0x1p-16f) continue;
        const uint32_t n = (word >> (4 * i)) & 15u;
        const uint32_t below = d[i] > 0.f ? n : n - 1u;  // the quotient is next to below + 1/2
        const double side = fma(-(static_cast<double>(below) + 0.5), static_cast<double>(scale),
                                static_cast<double>(x[i]) - low);
        const uint32_t code = below + (side > 0.0 || (side == 0.0 && (below & 1u)) ? 1u : 0u);
        word = (word & ~(15u << (4 * i))) | (code << (4 * i));
      }
    }
  }
  const bool odd = (w & 1) != 0;
  if constexpr (V) {
    // V: halves g = 2 t (low 16 bits) and 2 t + 1 of group w. The lane of an even
    // w keeps half 2 t and gets that of w + 1; the odd one keeps 2 t + 1.
    const uint32_t other = __shfl_xor_sync(0xffffffffu, word, 4);
    word = odd ? __byte_perm(other, word, 0x7632) : __byte_perm(word, other, 0x5410);
  }
  // Scales and lows in 32-bit words too: the lane of an even w stores the scales of
  // its pair of groups, that of the odd one the lows.
  const uint32_t sb = __half_as_ushort(scale_h), lb = __half_as_ushort(lo_h);
  const uint32_t traded = __shfl_xor_sync(0xffffffffu, odd ? sb : lb, 4);
  const uint32_t par = odd ? __byte_perm(traded, lb, 0x5410) : __byte_perm(sb, traded, 0x5410);
  if (!real) return;
  *reinterpret_cast<uint32_t*>(dst + 4 * word_of<D, V>(w, t)) = word;
  if (t == 0)
    *reinterpret_cast<uint32_t*>(dst + R::CODES + (odd ? 2 * R::NG : 0) + 4 * (w / 2)) = par;
}

// A lane takes its 8 values of K and of V of one (token, head): the slot and its
// row in the cache are found once for both. Mostly bound by its instructions (330 for
// the two, half of them the codes, 0.75 issued a cycle): 32768 tokens of 32 heads, d 128, bf16, B200:
// 200 us for 705 MB (3.5 TB/s; six CTAs per SM, 209 with five); with 64-bit divisions and
// one tensor per thread 628.
template <int D, typename T>
__global__ void __launch_bounds__(256, 6) kv4_append_kernel(const Kv4CopyParams p) {
  using R = Kv4Row<D>;
  constexpr int LPR = D / 8;  // lanes per row
  const int lane_row = threadIdx.x % LPR;
  const int w = lane_row / 4, t = lane_row % 4;
  const unsigned int row = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
  long long at = 0;
  bool real = row < p.rows;
  if (real) {
    const unsigned int token = p.by_hkv.quotient(row);
    const unsigned int head = row - token * p.hkv;
    const long long slot = p.slots[token];
    k = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.src[0]) +
                                        token * p.token_stride[0] + head * p.head_stride[0] +
                                        lane_row * 8);
    v = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.src[1]) +
                                        token * p.token_stride[1] + head * p.head_stride[1] +
                                        lane_row * 8);
    if (slot >= p.num_slots)
      report_status(p.status, 2u /* ATTN_DEVICE_BAD_BLOCK */, kSiteAppendSlot);
    real = slot >= 0 && slot < p.num_slots;
    if (real) at = cache_row(p, slot, static_cast<int>(head));
  }
  append_row<D, T, false>(static_cast<uint8_t*>(p.dst[0]) + at * R::BYTES, k, real, w, t);
  append_row<D, T, true>(static_cast<uint8_t*>(p.dst[1]) + at * R::BYTES, v, real, w, t);
  if (real && lane_row == 0 && p.weights != nullptr) p.weights[at] = 0.f;
}

// The inverse for one lane of a row: its 8 values from the word of their codes and
// their group's scale and low.
template <typename T>
__device__ __forceinline__ uint4 values_of(uint32_t v, uint16_t scale_h, uint16_t low_h) {
  const uint32_t scale_bits = scale_h * 0x10001u, low_bits = low_h * 0x10001u;
  uint32_t out[4];
  if constexpr (std::is_same<T, __half>::value) {
    // low + scale * code in one fp16 fma is the value rounded once. Codes j and
    // j + 4 come together: 1024 + code by its bits, less 1024.
    uint32_t y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t n = ((v >> (4 * j)) & 0x000F000Fu) | 0x64006400u;
      const __half2 code = __hadd2(*reinterpret_cast<const __half2*>(&n), __float2half2_rn(-1024.f));
      const __half2 x = __hfma2(code, *reinterpret_cast<const __half2*>(&scale_bits),
                                *reinterpret_cast<const __half2*>(&low_bits));
      y[j] = *reinterpret_cast<const uint32_t*>(&x);
    }
    out[0] = __byte_perm(y[0], y[1], 0x5410);
    out[1] = __byte_perm(y[2], y[3], 0x5410);
    out[2] = __byte_perm(y[0], y[1], 0x7632);
    out[3] = __byte_perm(y[2], y[3], 0x7632);
  } else {
    // In fp32, 16^j code (code j where it stands in the word, below 2^23) by its
    // bits and with the scale times 16^-j; codes 5 to 7 from the word shifted.
    const float scale = __half2float(__ushort_as_half(scale_h));
    const float low = __half2float(__ushort_as_half(low_h));
    const uint64_t low2 = f2_pack(low, low), minus2 = f2_pack(-8388608.f, -8388608.f);
    const uint32_t top = v >> 20;
    const uint32_t bits[8] = {v & 0xFu,     v & 0xF0u,  v & 0xF00u, v & 0xF000u,
                              v & 0xF0000u, top & 0xFu, top & 0xF0u, top & 0xF00u};
    constexpr float down[8] = {1.f,      0x1p-4f, 0x1p-8f, 0x1p-12f,
                               0x1p-16f, 1.f,     0x1p-4f, 0x1p-8f};
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const uint64_t n = f2_add(f2_pack(__uint_as_float(0x4B000000u | bits[e]),
                                        __uint_as_float(0x4B000000u | bits[e + 1])), minus2);
      const uint64_t s2 = f2_pack(scale * down[e], scale * down[e + 1]);
      float x0, x1;
      f2_unpack(f2_fma(s2, n, low2), x0, x1);
      out[e / 2] = pack2<T>(x0, x1);
    }
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

// Lane (w, t) of a row reads the word of its codes (of V the word that it traded
// when writing) and its group's scale and low of K and of V. Slots below 0 read as
// zeros. The shape above: 142 us (5.0 TB/s).
template <int D, typename T>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4CopyParams p) {
  using R = Kv4Row<D>;
  constexpr int LPR = D / 8;
  const int lane_row = threadIdx.x % LPR;
  const int w = lane_row / 4, t = lane_row % 4;
  const unsigned int row = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  uint32_t word[2] = {0u, 0u};
  uint16_t scale[2] = {0, 0}, low[2] = {0, 0};
  if (row < p.rows) {
    const unsigned int token = p.by_hkv.quotient(row);
    const long long slot = p.slots[token];
    if (slot >= p.num_slots)
      report_status(p.status, 2u /* ATTN_DEVICE_BAD_BLOCK */, kSiteReadSlot);
    else if (slot >= 0) {
      const long long at =
          cache_row(p, slot, static_cast<int>(row - token * p.hkv)) * R::BYTES;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint8_t* src = static_cast<const uint8_t*>(p.src[i]) + at;
        const uint16_t* par = reinterpret_cast<const uint16_t*>(src + R::CODES);
        word[i] = *reinterpret_cast<const uint32_t*>(
            src + 4 * (i == 0 ? word_of<D, false>(w, t) : word_of<D, true>(w, t)));
        scale[i] = par[w];
        low[i] = par[R::NG + w];
      }
    }
  }
  const uint32_t other = __shfl_xor_sync(0xffffffffu, word[1], 4);
  word[1] = (w & 1) ? __byte_perm(other, word[1], 0x7632) : __byte_perm(word[1], other, 0x5410);
  if (row >= p.rows) return;
  const size_t to = static_cast<size_t>(row) * D + lane_row * 8;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    *reinterpret_cast<uint4*>(static_cast<T*>(p.dst[i]) + to) =
        values_of<T>(word[i], scale[i], low[i]);
}

Kv4CopyParams params_of(const Kv4CopyArgs& a, const LaunchCtx& ctx) {
  Kv4CopyParams p;
  for (int i = 0; i < 2; ++i) {
    p.token_stride[i] = a.token_stride[i];
    p.head_stride[i] = a.head_stride[i];
  }
  p.slots = reinterpret_cast<const long long*>(a.slots);
  p.weights = a.weights;
  p.status = ctx.status;
  p.rows = static_cast<unsigned int>(a.tokens * a.hkv);
  p.num_slots = a.num_blocks * a.bs;
  p.hkv = static_cast<int>(a.hkv);
  p.bs = static_cast<int>(a.bs);
  p.by_hkv = FastDiv(a.hkv);
  p.by_bs = FastDiv(a.bs);
  p.narrow = a.num_blocks <= 0x7fffffffLL / (a.bs * a.hkv) ? 1 : 0;
  return p;
}

unsigned grid_of(const Kv4CopyArgs& a) {
  const int64_t rows_per_cta = 256 / (a.d / 8);
  return static_cast<unsigned>((a.tokens * a.hkv + rows_per_cta - 1) / rows_per_cta);
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4CopyArgs& a, const LaunchCtx& ctx) {
  Kv4CopyParams p = params_of(a, ctx);
  p.src[0] = a.k;
  p.src[1] = a.v;
  p.dst[0] = a.k_cache;
  p.dst[1] = a.v_cache;
  const unsigned grid = grid_of(a);
  if (a.d == 64) {
    if (a.bf16) kv4_append_kernel<64, __nv_bfloat16><<<grid, 256, 0, ctx.stream>>>(p);
    else kv4_append_kernel<64, __half><<<grid, 256, 0, ctx.stream>>>(p);
  } else {
    if (a.bf16) kv4_append_kernel<128, __nv_bfloat16><<<grid, 256, 0, ctx.stream>>>(p);
    else kv4_append_kernel<128, __half><<<grid, 256, 0, ctx.stream>>>(p);
  }
  return cudaGetLastError();
}

cudaError_t launch_kv4_read(const Kv4CopyArgs& a, const LaunchCtx& ctx) {
  Kv4CopyParams p = params_of(a, ctx);
  p.src[0] = a.k_cache;
  p.src[1] = a.v_cache;
  p.dst[0] = a.k;
  p.dst[1] = a.v;
  const unsigned grid = grid_of(a);
  if (a.d == 64) {
    if (a.bf16) kv4_read_kernel<64, __nv_bfloat16><<<grid, 256, 0, ctx.stream>>>(p);
    else kv4_read_kernel<64, __half><<<grid, 256, 0, ctx.stream>>>(p);
  } else {
    if (a.bf16) kv4_read_kernel<128, __nv_bfloat16><<<grid, 256, 0, ctx.stream>>>(p);
    else kv4_read_kernel<128, __half><<<grid, 256, 0, ctx.stream>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace fab
