// Decode attention of one query token per sequence over the 4-bit paged cache
// (row layout: kv4.cuh), split over the context and merged like the fp16 decode
// (decode.cu): scores in log2 units, a running maximum and sum, one fp32
// (o, m, l) part per split.
#include <algorithm>

#include "kv4.cuh"
#include "launch.h"

namespace fab {
namespace {

enum : unsigned int { kSiteKv4Block = 221 };

struct Kv4DecParams {
  const void* q;          // [batch, hq, D] fp16 or bf16
  const uint8_t* kc;      // [num_blocks, hkv, bs, row]
  const uint8_t* vc;
  const int* bt;
  const int* ctx;
  float* o_part;          // [batch * hq, num_splits, D]
  float* m_part;          // [batch * hq, num_splits]
  float* l_part;
  float* scores;          // [batch, hkv, max_ctx, gp] log2-unit scores, or null
  DeviceStatus* status;
  int batch, hq, hkv, group, gp, bs, max_blocks, num_blocks, partition, num_splits, max_ctx;
  float scale_log2;
};

// One CTA per (split, kv head, sequence): its four warps take tokens in turn,
// lane i holding dims i, i + 32, ... of every row.
template <int D, typename T>
__global__ void __launch_bounds__(128) kv4_decode_kernel(const Kv4DecParams p) {
  using R = Kv4Row<D>;
  constexpr int NG = R::NG;
  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int ctx = min(max(p.ctx[b], 0), p.max_ctx);
  const int t0 = split * p.partition, t1 = min(ctx, t0 + p.partition);
  if (t0 >= ctx) return;
  float q[8][NG], acc[8][NG], m[8], l[8];
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int w = 0; w < NG; ++w) {
      acc[g][w] = 0.f;
      q[g][w] = g < p.group ? to_f32(static_cast<const T*>(p.q)[(static_cast<size_t>(b) * p.hq +
                                  kvh * p.group + g) * D + 32 * w + lane]) * p.scale_log2 : 0.f;
    }
  }
  for (int t = t0 + warp; t < t1; t += 4) {
    int page = p.bt[static_cast<size_t>(b) * p.max_blocks + t / p.bs];
    if (page < 0 || page >= p.num_blocks) {
      if (lane == 0) report_status(p.status, 2u, kSiteKv4Block);
      page = 0;
    }
    const size_t off =
        ((static_cast<size_t>(page) * p.hkv + kvh) * p.bs + t % p.bs) * R::BYTES;
    const uint8_t* kr = p.kc + off;
    const uint8_t* vr = p.vc + off;
    float kx[NG], vx[NG];
#pragma unroll
    for (int w = 0; w < NG; ++w) {
      const uint32_t kw = reinterpret_cast<const uint32_t*>(kr)[(lane / 8) * NG + w];
      const uint32_t vw = reinterpret_cast<const uint16_t*>(vr)[(lane / 4) * NG + w];
      const __half* kp = reinterpret_cast<const __half*>(kr + R::CODES);
      const __half* vp = reinterpret_cast<const __half*>(vr + R::CODES);
      kx[w] = fmaf(__half2float(kp[w]), static_cast<float>((kw >> (4 * (lane % 8))) & 15u),
                   __half2float(kp[NG + w]));
      vx[w] = fmaf(__half2float(vp[w]), static_cast<float>((vw >> (4 * (lane % 4))) & 15u),
                   __half2float(vp[NG + w]));
    }
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      if (g >= p.group) break;
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < NG; ++w) s = fmaf(q[g][w], kx[w], s);
      s = warp_sum(s);
      if (p.scores != nullptr && lane == 0)
        p.scores[((static_cast<size_t>(b) * p.hkv + kvh) * p.max_ctx + t) * p.gp + g] = s;
      const float mn = fmaxf(m[g], s);
      const float alpha = exp2f(m[g] - mn), e = exp2f(s - mn);
      l[g] = l[g] * alpha + e;
      m[g] = mn;
#pragma unroll
      for (int w = 0; w < NG; ++w) acc[g][w] = fmaf(e, vx[w], acc[g][w] * alpha);
    }
  }
  __shared__ float so[4][8][D], sm[4][8], sl[4][8];
#pragma unroll
  for (int g = 0; g < 8; ++g) {
#pragma unroll
    for (int w = 0; w < NG; ++w) so[warp][g][32 * w + lane] = acc[g][w];
    sm[warp][g] = m[g];
    sl[warp][g] = l[g];
  }
  __syncthreads();
  for (int g = warp; g < p.group; g += 4) {
    const float mx = fmaxf(fmaxf(sm[0][g], sm[1][g]), fmaxf(sm[2][g], sm[3][g]));
    float a[4], den = 0.f;
    for (int i = 0; i < 4; ++i) {
      a[i] = sm[i][g] == -INFINITY ? (sl[i][g] != sl[i][g] ? 1.f : 0.f) : exp2f(sm[i][g] - mx);
      den += a[i] * sl[i][g];
    }
    const size_t pr = (static_cast<size_t>(b) * p.hq + kvh * p.group + g) * p.num_splits + split;
    for (int w = 0; w < NG; ++w) {
      float num = 0.f;
      for (int i = 0; i < 4; ++i) num += a[i] * so[i][g][32 * w + lane];
      p.o_part[pr * D + 32 * w + lane] = num / den;
    }
    if (lane == 0) {
      // A part whose scores are all NaN has no maximum, yet is not an empty one.
      p.m_part[pr] = den != den ? fmaxf(mx, 0.f) : mx;
      p.l_part[pr] = den;
    }
  }
}

size_t align256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

struct Workspace {
  float *o, *m, *l, *scores;
  size_t bytes;
};

Workspace carve(void* base, int64_t rows, int64_t d, int64_t splits, size_t score_bytes) {
  uint8_t* b = static_cast<uint8_t*>(base);
  const size_t ob = align256(static_cast<size_t>(rows) * splits * d * 4);
  const size_t ml = align256(static_cast<size_t>(rows) * splits * 4);
  Workspace w;
  w.o = reinterpret_cast<float*>(b);
  w.m = reinterpret_cast<float*>(b + ob);
  w.l = reinterpret_cast<float*>(b + ob + ml);
  w.scores = reinterpret_cast<float*>(b + ob + 2 * ml);
  w.bytes = ob + 2 * ml + align256(score_bytes);
  return w;
}

}  // namespace

size_t kv4_decode_workspace_bytes(int64_t batch, int64_t hq, int64_t hkv, int64_t d, int64_t max_ctx,
                                  int64_t partition, bool weights) {
  const int64_t splits = (max_ctx + partition - 1) / partition;
  return carve(nullptr, batch * hq, d, splits,
               weights ? score_bytes(batch, hkv, hq / hkv, max_ctx) : 0).bytes;
}

cudaError_t launch_kv4_decode(const Kv4DecodeArgs& a, const LaunchCtx& ctx) {
  const int64_t splits = (a.max_ctx + a.partition - 1) / a.partition;
  const int64_t group = a.hq / a.hkv;
  if (splits == 0)
    return cudaMemsetAsync(a.out, 0, static_cast<size_t>(a.batch) * a.hq * a.d * 2, ctx.stream);
  Workspace w = carve(a.workspace, a.batch * a.hq, a.d, splits,
                      a.weights != nullptr ? score_bytes(a.batch, a.hkv, group, a.max_ctx) : 0);
  Kv4DecParams p;
  p.q = a.q;
  p.kc = static_cast<const uint8_t*>(a.k_cache);
  p.vc = static_cast<const uint8_t*>(a.v_cache);
  p.bt = a.block_tables;
  p.ctx = a.context_lens;
  p.o_part = w.o;
  p.m_part = w.m;
  p.l_part = w.l;
  p.scores = a.weights != nullptr ? w.scores : nullptr;
  p.status = ctx.status;
  p.batch = static_cast<int>(a.batch);
  p.hq = static_cast<int>(a.hq);
  p.hkv = static_cast<int>(a.hkv);
  p.group = static_cast<int>(group);
  p.gp = static_cast<int>(score_heads(group));
  p.bs = static_cast<int>(a.bs);
  p.max_blocks = static_cast<int>(a.max_blocks);
  p.num_blocks = static_cast<int>(a.num_blocks);
  p.partition = static_cast<int>(a.partition);
  p.num_splits = static_cast<int>(splits);
  p.max_ctx = static_cast<int>(a.max_ctx);
  p.scale_log2 = a.scale * kLog2e;
  const dim3 grid(static_cast<unsigned>(splits), static_cast<unsigned>(a.hkv),
                  static_cast<unsigned>(a.batch));
  if (a.d == 64) {
    if (a.bf16) kv4_decode_kernel<64, __nv_bfloat16><<<grid, 128, 0, ctx.stream>>>(p);
    else kv4_decode_kernel<64, __half><<<grid, 128, 0, ctx.stream>>>(p);
  } else {
    if (a.bf16) kv4_decode_kernel<128, __nv_bfloat16><<<grid, 128, 0, ctx.stream>>>(p);
    else kv4_decode_kernel<128, __half><<<grid, 128, 0, ctx.stream>>>(p);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  DecodePartsArgs f{w.o, w.m, w.l, a.context_lens, a.batch, a.hq, a.hkv, a.d, a.partition, splits,
                    false, a.out, a.bf16};
  e = launch_decode_merge(f, ctx);
  if (e != cudaSuccess || a.weights == nullptr) return e;
  return launch_add_weights({w.scores, w.m, w.l, a.block_tables, a.context_lens, a.weights, a.batch,
                             a.hq, a.hkv, a.bs, a.num_blocks, a.max_blocks, a.max_ctx, a.partition,
                             splits}, ctx);
}

}  // namespace fab
