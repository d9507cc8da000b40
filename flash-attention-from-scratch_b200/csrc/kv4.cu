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
  long long rows;             // tokens * hkv
  long long num_slots;        // num_blocks * bs
  int hkv, bs;
};

// Byte offset of row (slot, head) in a cache of rows of `row` bytes.
__device__ __forceinline__ long long row_offset(long long slot, int head, int hkv, int bs, int row) {
  const long long page = slot / bs;
  return ((page * hkv + head) * bs + (slot - page * bs)) * row;
}

// Four lanes per group, each with 8 of its 32 values in one 16-byte load: lane
// t of the group makes exactly the row's 32-bit K word (t, w); of V it makes the
// 16-bit words g = 2 t and 2 t + 1 of group w, and trades one of them with the
// lane of group w ^ 1, so that every lane stores one 32-bit word and a row's
// codes are one contiguous store of the warp.
template <int D, typename T>
__global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4CopyParams p) {
  using R = Kv4Row<D>;
  constexpr int LPR = D / 8;  // lanes per row
  const int which = blockIdx.y;
  const int lane_row = threadIdx.x % LPR;
  const int w = lane_row / 4, t = lane_row % 4;
  const long long row = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) / LPR;
  const bool real = row < p.rows;
  long long slot = -1;
  int head = 0;
  float x[8];
  if (real) {
    const long long token = row / p.hkv;
    head = static_cast<int>(row - token * p.hkv);
    slot = p.slots[token];
    if (slot >= p.num_slots) {
      report_status(p.status, 2u /* ATTN_DEVICE_BAD_BLOCK */, kSiteAppendSlot);
      slot = -1;
    }
    const T* src = static_cast<const T*>(p.src[which]) + token * p.token_stride[which] +
                   head * p.head_stride[which] + lane_row * 8;
    const uint4 raw = *reinterpret_cast<const uint4*>(src);
    const T* v = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
  }
  float lo = x[0], hi = x[0];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    bad = bad || !(fabsf(x[i]) <= 65504.f);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    bad = __shfl_xor_sync(0xffffffffu, static_cast<int>(bad), o) || bad;
  }
  __half lo_h = __float2half_rn(lo);
  const float low = __half2float(lo_h);
  __half scale_h = __float2half_rn(__fdiv_rn(hi - low, 15.f));
  if (bad) lo_h = scale_h = __ushort_as_half(0x7fff);  // NaN
  const float scale = __half2float(scale_h);
  uint32_t word = 0;
  if (scale > 0.f) {
    const float inv = 1.f / scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // The quotient to a few fp32 roundings; where that could decide between
      // two codes (next to a half), in 64 bits.
      float r = fminf(fmaxf((x[i] - low) * inv, 0.f), 15.f);
      float n = rintf(r);
      if (fabsf(r - n) > 0.5f - 0x1p-16f) {
        const double q = (static_cast<double>(x[i]) - low) / static_cast<double>(scale);
        n = static_cast<float>(fmin(fmax(rint(q), 0.0), 15.0));
      }
      word |= static_cast<uint32_t>(n) << (4 * i);
    }
  }
  if (which == 1) {
    // V: halves g = 2 t (low 16 bits) and 2 t + 1 of group w. The lane of an even
    // w keeps half 2 t and gets that of w + 1; the odd one keeps 2 t + 1.
    const uint32_t other = __shfl_xor_sync(0xffffffffu, word, 4);
    word = (w & 1) == 0 ? __byte_perm(word, other, 0x5410) : __byte_perm(other, word, 0x7632);
  }
  if (slot < 0) return;
  uint8_t* dst = static_cast<uint8_t*>(p.dst[which]) + row_offset(slot, head, p.hkv, p.bs, R::BYTES);
  const int word_at = which == 0 ? t * R::NG + w : ((2 * t + (w & 1)) * R::NG + (w & ~1)) / 2;
  *reinterpret_cast<uint32_t*>(dst + 4 * word_at) = word;
  if (t < 2)
    reinterpret_cast<__half*>(dst + R::CODES)[t * R::NG + w] = t == 0 ? scale_h : lo_h;
  if (which == 0 && lane_row == 0 && p.weights != nullptr) {
    const long long page = slot / p.bs;
    p.weights[(page * p.hkv + head) * p.bs + (slot - page * p.bs)] = 0.f;
  }
}

// The inverse: lane (w, t) of a row reads the word(s) of its 8 values and their
// group's scale and low, and writes 16 bytes. Slots below 0 read as zeros.
template <int D, typename T>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4CopyParams p) {
  using R = Kv4Row<D>;
  constexpr int LPR = D / 8;
  const int which = blockIdx.y;
  const int lane_row = threadIdx.x % LPR;
  const int w = lane_row / 4, t = lane_row % 4;
  const long long row = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) / LPR;
  if (row >= p.rows) return;
  const long long token = row / p.hkv;
  const int head = static_cast<int>(row - token * p.hkv);
  long long slot = p.slots[token];
  if (slot >= p.num_slots) {
    report_status(p.status, 2u /* ATTN_DEVICE_BAD_BLOCK */, kSiteReadSlot);
    slot = -1;
  }
  uint4 out = make_uint4(0u, 0u, 0u, 0u);
  if (slot >= 0) {
    const uint8_t* src =
        static_cast<const uint8_t*>(p.src[which]) + row_offset(slot, head, p.hkv, p.bs, R::BYTES);
    const __half* par = reinterpret_cast<const __half*>(src + R::CODES);
    const float scale = __half2float(par[w]), low = __half2float(par[R::NG + w]);
    uint32_t word;
    if (which == 0) {
      word = *reinterpret_cast<const uint32_t*>(src + 4 * (t * R::NG + w));
    } else {
      const uint16_t* half = reinterpret_cast<const uint16_t*>(src);
      word = half[2 * t * R::NG + w] | (static_cast<uint32_t>(half[(2 * t + 1) * R::NG + w]) << 16);
    }
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf(scale, static_cast<float>((word >> (4 * i)) & 15u), low);
    out = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]),
                     pack2<T>(x[6], x[7]));
  }
  T* dst = static_cast<T*>(p.dst[which]) + row * D + lane_row * 8;
  *reinterpret_cast<uint4*>(dst) = out;
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
  p.rows = a.tokens * a.hkv;
  p.num_slots = a.num_blocks * a.bs;
  p.hkv = static_cast<int>(a.hkv);
  p.bs = static_cast<int>(a.bs);
  return p;
}

dim3 grid_of(const Kv4CopyArgs& a) {
  const int64_t rows_per_cta = 256 / (a.d / 8);
  return dim3(static_cast<unsigned>((a.tokens * a.hkv + rows_per_cta - 1) / rows_per_cta), 2);
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4CopyArgs& a, const LaunchCtx& ctx) {
  Kv4CopyParams p = params_of(a, ctx);
  p.src[0] = a.k;
  p.src[1] = a.v;
  p.dst[0] = a.k_cache;
  p.dst[1] = a.v_cache;
  const dim3 grid = grid_of(a);
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
  const dim3 grid = grid_of(a);
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
