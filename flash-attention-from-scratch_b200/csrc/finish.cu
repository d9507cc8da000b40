// The end of a split decode launch, in one kernel: the fp32 (o, m, l) parts of a
// row are merged,
//     M = max_s m_s,  L = sum_s l_s 2^(m_s - M),  o = sum_s l_s 2^(m_s - M) o_s / L,
// and, where the decode left every token's score s (log2 units), the token's
// attention weight 2^(s - M) / L, summed over the query heads of its kv head, is
// added to its slot's total. One kernel, because a short call is bound by its
// launches: the CTAs that add weights find M and L from the parts themselves
// instead of waiting for a merge.
#include <algorithm>

#include "kv4.cuh"
#include "launch.h"

namespace fab {
namespace {

enum : unsigned int { kSiteWeightBlock = 241 };

struct FinishParams {
  const float* o;
  const float* m;
  const float* l;
  const int* ctx;
  const int* first;
  const float* scores;
  float* weights;
  const int* bt;
  void* out;
  DeviceStatus* status;
  unsigned int workers;
  int partition, parts;
  int batch, hq, hkv, group, gp, bs, num_blocks, max_blocks, max_ctx;
  int merge_blocks;  // CTAs [0, merge_blocks) merge, the others add weights
  int add_chunks;    // CTAs per (sequence, kv head) that add
  FastDiv by_bs;
};

// The parts of one (sequence, kv head) pair: part s of query head g is at
// base + s * stride + g * head. An empty sequence has none.
struct Parts {
  long long base, stride, head;
  int count;
};

__device__ __forceinline__ Parts parts_of(const FinishParams& p, int b, int kvh, int ctx) {
  Parts r;
  if (p.first == nullptr) {
    r.count = min((ctx + p.partition - 1) / p.partition, p.parts);
    r.base = (static_cast<long long>(b) * p.hq + kvh * p.group) * p.parts;
    r.stride = 1;
    r.head = p.parts;
    return r;
  }
  const int n = p.first[b + 1] - p.first[b];
  if (n == 0) return {0, 0, 0, 0};
  const Runs runs(static_cast<unsigned int>(p.first[p.batch]) * p.hkv, p.workers);
  const unsigned int s0 = static_cast<unsigned int>(p.first[b]) * p.hkv + kvh * n;
  const unsigned int i0 = runs.of(s0), i1 = runs.of(s0 + n - 1);
  r.count = static_cast<int>(i1 - i0 + 1);
  r.base = (static_cast<long long>(i0) + b * p.hkv + kvh) * p.group;
  r.stride = p.group;
  r.head = 1;
  return r;
}

// Threads of a CTA.
template <int WPR>
constexpr int kThreads = WPR == 32 ? 1024 : 256;

// WPR warps per row (a power of two) merge: lane owns D / 32 columns; each warp folds
// chunks of 8 parts into a running (max, sum, numerator), and the warps of a row
// combine in shared memory. A chunk is one round trip to memory, so rows with many
// parts (few rows, a long context) take more warps.
template <int D, int WPR, typename T>
__device__ void merge_row(const FinishParams& p, long long row, bool live, const Parts& r, int g) {
  constexpr int DV = D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % WPR;
  float mw = -INFINITY, den = 0.f, num[DV];
#pragma unroll
  for (int j = 0; j < DV; ++j) num[j] = 0.f;
  if (live) {
    const long long at = r.base + g * r.head;
    const int per = (r.count + WPR - 1) / WPR;
    const int begin = min(r.count, sub * per), end = min(r.count, begin + per);
    for (int s0 = begin; s0 < end; s0 += 8) {
      const int cnt = min(8, end - s0);
      // Lane u holds m and l of part s0 + u % 8.
      const bool have = (lane & 7) < cnt;
      const long long su = at + (s0 + (lane & 7)) * r.stride;
      const float mu = have ? p.m[su] : -INFINITY;
      const float lu = have ? p.l[su] : 0.f;
      float v[8][DV];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float* src = p.o + (at + (s0 + u) * r.stride) * D + lane * DV;
        if (u < cnt) {
          if constexpr (DV == 4) {
            const float4 x = *reinterpret_cast<const float4*>(src);
            v[u][0] = x.x; v[u][1] = x.y; v[u][2] = x.z; v[u][3] = x.w;
          } else {
            const float2 x = *reinterpret_cast<const float2*>(src);
            v[u][0] = x.x; v[u][1] = x.y;
          }
        } else {
#pragma unroll
          for (int j = 0; j < DV; ++j) v[u][j] = 0.f;
        }
      }
      float mn = mu;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mn = fmaxf(mw, mn);
      const float alpha = mw == -INFINITY ? 0.f : fast_exp2(mw - mn);
      const float wu = have ? lu * fast_exp2(mu - mn) : 0.f;
      float ws = wu;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
      den = den * alpha + ws;
#pragma unroll
      for (int j = 0; j < DV; ++j) num[j] *= alpha;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float w = __shfl_sync(0xffffffffu, wu, u);
#pragma unroll
        for (int j = 0; j < DV; ++j) num[j] = fmaf(w, v[u][j], num[j]);
      }
      mw = mn;
    }
  }
  if constexpr (WPR > 1) {
    __shared__ float red[kThreads<WPR> / 32][D + 2];
    const int row0 = warp - sub;  // the row's first warp
#pragma unroll
    for (int j = 0; j < DV; ++j) red[warp][lane * DV + j] = num[j];
    if (lane == 0) {
      red[warp][D] = den;
      red[warp][D + 1] = mw;
    }
    __syncthreads();
    if (!live || sub != 0) return;
    float big = mw;
    for (int w = 1; w < WPR; ++w) big = fmaxf(big, red[row0 + w][D + 1]);
    den = 0.f;
#pragma unroll
    for (int j = 0; j < DV; ++j) num[j] = 0.f;
    for (int w = 0; w < WPR; ++w) {
      const float mx = red[row0 + w][D + 1];
      if (mx == -INFINITY) continue;  // a warp without parts
      const float a = fast_exp2(mx - big);
      den = fmaf(a, red[row0 + w][D], den);
#pragma unroll
      for (int j = 0; j < DV; ++j) num[j] = fmaf(a, red[row0 + w][lane * DV + j], num[j]);
    }
  }
  if (!live) return;
  // An empty sequence has no part: zeros.
  const float inv = r.count == 0 ? 0.f : 1.f / den;
  uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + row * D + lane * DV);
#pragma unroll
  for (int j = 0; j < DV; j += 2) dst[j / 2] = pack2<T>(num[j] * inv, num[j + 1] * inv);
}

constexpr int kAddTokens = 1024;  // tokens a CTA adds at a time

// The totals of up to kAddTokens tokens of one (sequence, kv head), GP scores a
// token. A CTA's scores are on their way while it finds M and L of its query heads.
template <int GP, int THREADS>
__device__ void add_weights(const FinishParams& p) {
  constexpr int U = kAddTokens / THREADS;  // tokens per thread
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int at = blockIdx.x - p.merge_blocks;
  const int pair = at / p.add_chunks, chunk = at - pair * p.add_chunks;
  const int b = pair / p.hkv, kvh = pair - b * p.hkv;
  const int ctx = min(max(p.ctx[b], 0), p.max_ctx);
  // Lengths are below 2^31, a chunk past the end of one below 2^32.
  unsigned int t0 = static_cast<unsigned int>(chunk) * kAddTokens;
  const unsigned int stride = static_cast<unsigned int>(p.add_chunks) * kAddTokens;
  const unsigned int end = static_cast<unsigned int>(ctx);
  if (t0 >= end) return;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float mx[8], inv[8];
  const int* bt = p.bt + static_cast<size_t>(b) * p.max_blocks;
  const float* sc = p.scores + static_cast<size_t>(pair) * p.max_ctx * GP;
  float* totals = p.weights + static_cast<size_t>(kvh) * p.bs;
  const unsigned int page_stride = static_cast<unsigned int>(p.hkv) * p.bs;
  float s[U][GP];
  int page[U];
  auto load = [&]() {
    const float* src = sc + (static_cast<size_t>(t0) + threadIdx.x) * GP;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned int t = t0 + u * THREADS + threadIdx.x;
      if (t >= end) break;
      const float* at = src + u * THREADS * GP;
      if constexpr (GP == 1) {
        s[u][0] = *at;
      } else if constexpr (GP == 2) {
        const float2 x = *reinterpret_cast<const float2*>(at);
        s[u][0] = x.x; s[u][1] = x.y;
      } else {
#pragma unroll
        for (int i = 0; i < GP; i += 4) {
          const float4 x = *reinterpret_cast<const float4*>(at + i);
          s[u][i] = x.x; s[u][i + 1] = x.y; s[u][i + 2] = x.z; s[u][i + 3] = x.w;
        }
      }
      page[u] = bt[p.by_bs.quotient(t)];
    }
  };
  load();
  const Parts r = parts_of(p, b, kvh, ctx);
  if (warp < p.group) {
    const long long base = r.base + warp * r.head;
    float big = -INFINITY, sum = 0.f;
    for (int i = lane; i < r.count; i += 32) {
      const float m = p.m[base + i * r.stride], l = p.l[base + i * r.stride];
      const float mn = fmaxf(big, m);
      sum = (big == -INFINITY ? 0.f : sum * exp2f(big - mn)) + l * exp2f(m - mn);
      big = mn;
    }
    const float all = warp_max(big);
    sum = warp_sum(big == -INFINITY ? 0.f : sum * exp2f(big - all));
    if (lane == 0) {
      mx[warp] = all;
      inv[warp] = 1.f / sum;
    }
  }
  __syncthreads();
  float mh[GP], ih[GP];
#pragma unroll
  for (int g = 0; g < GP; ++g) {
    // Heads past the group (GP is a power of two) weigh nothing.
    mh[g] = g < p.group ? mx[g] : 0.f;
    ih[g] = g < p.group ? inv[g] : 0.f;
  }
  for (;;) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned int t = t0 + u * THREADS + threadIdx.x;
      if (t >= end) break;
      float w = 0.f;
#pragma unroll
      for (int g = 0; g < GP; ++g)
        if (g < p.group) w = fmaf(fast_exp2(s[u][g] - mh[g]), ih[g], w);
      if (static_cast<unsigned>(page[u]) >= static_cast<unsigned>(p.num_blocks)) {
        report_status(p.status, 2u /* ATTN_DEVICE_BAD_BLOCK */, kSiteWeightBlock);
        continue;
      }
      // A page can stand in several sequences (a shared prefix): their adds all count.
      atomicAdd(totals + static_cast<unsigned long long>(static_cast<unsigned>(page[u])) * page_stride +
                    (t - p.by_bs.quotient(t) * p.bs), w);
    }
    t0 += stride;
    if (t0 >= end) break;
    load();
  }
}

// Launched as a programmatic dependent of the decode: it waits for that launch's
// end before it reads what the decode wrote (lengths are an input of both).
template <int D, int WPR, typename T>
__global__ void __launch_bounds__(kThreads<WPR>) finish_kernel(const FinishParams p) {
  constexpr int THREADS = kThreads<WPR>;
  const int warp = threadIdx.x >> 5;
  if (static_cast<int>(blockIdx.x) < p.merge_blocks) {
    const long long row = static_cast<long long>(blockIdx.x) * (THREADS / 32 / WPR) + warp / WPR;
    bool live = row < static_cast<long long>(p.batch) * p.hq;
    Parts r = {0, 0, 0, 0};
    const int b = live ? static_cast<int>(row / p.hq) : 0;
    const int head = live ? static_cast<int>(row - static_cast<long long>(b) * p.hq) : 0;
    const int kvh = head / p.group, g = head - kvh * p.group;
    const int ctx = min(max(p.ctx[b], 0), p.max_ctx);  // an input of the decode too
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (live) {
      r = parts_of(p, b, kvh, ctx);
      if (p.first != nullptr && r.count == 1) live = false;  // written by the decode
    }
    merge_row<D, WPR, T>(p, row, live, r, g);
    return;
  }
  switch (p.gp) {
    case 1: add_weights<1, THREADS>(p); break;
    case 2: add_weights<2, THREADS>(p); break;
    case 4: add_weights<4, THREADS>(p); break;
    default: add_weights<8, THREADS>(p); break;
  }
}

template <int D, int WPR, typename T>
cudaError_t launch(const FinishParams& p, unsigned grid, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads<WPR>);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, finish_kernel<D, WPR, T>, p);
}

template <int D, int WPR>
cudaError_t by_type(const FinishParams& p, unsigned grid, bool bf16, cudaStream_t stream) {
  return bf16 ? launch<D, WPR, __nv_bfloat16>(p, grid, stream)
              : launch<D, WPR, __half>(p, grid, stream);
}

template <int D>
cudaError_t by_warps(const FinishParams& p, unsigned grid, int wpr, bool bf16,
                     cudaStream_t stream) {
  return wpr == 32  ? by_type<D, 32>(p, grid, bf16, stream)
         : wpr == 8 ? by_type<D, 8>(p, grid, bf16, stream)
         : wpr == 4 ? by_type<D, 4>(p, grid, bf16, stream)
         : wpr == 2 ? by_type<D, 2>(p, grid, bf16, stream)
                    : by_type<D, 1>(p, grid, bf16, stream);
}

}  // namespace

int64_t score_heads(int64_t group) {
  int64_t gp = 1;
  while (gp < group) gp *= 2;
  return gp;
}

size_t score_bytes(int64_t batch, int64_t hkv, int64_t group, int64_t max_ctx) {
  return static_cast<size_t>(batch) * hkv * max_ctx * score_heads(group) * 4;
}

cudaError_t launch_finish(const FinishArgs& a, const LaunchCtx& ctx) {
  FinishParams p;
  p.o = a.o;
  p.m = a.m;
  p.l = a.l;
  p.ctx = a.context_lens;
  p.first = a.first;
  p.scores = a.scores;
  p.weights = a.weights;
  p.bt = a.block_tables;
  p.out = a.out;
  p.status = ctx.status;
  p.workers = static_cast<unsigned int>(a.workers);
  p.partition = static_cast<int>(a.partition);
  p.parts = static_cast<int>(a.parts);
  p.batch = static_cast<int>(a.batch);
  p.hq = static_cast<int>(a.hq);
  p.hkv = static_cast<int>(a.hkv);
  p.group = static_cast<int>(a.hq / a.hkv);
  p.gp = static_cast<int>(score_heads(p.group));
  p.bs = static_cast<int>(a.bs);
  p.by_bs = FastDiv(a.bs);
  p.num_blocks = static_cast<int>(a.num_blocks);
  p.max_blocks = static_cast<int>(a.max_blocks);
  p.max_ctx = static_cast<int>(a.max_ctx);
  const int64_t rows = a.batch * a.hq;
  // Warps per row by the parts a row can have: up to four chunks of 8 a warp; more warps
  // where few rows leave SMs idle meanwhile (4-bit decode, head_dim 128, 8 kv heads of 4
  // query heads, one / up to 8 warps a row, us: 8 x 1728 tokens 17.1 / 12.6, 16 x 1152
  // 15.6 / 14.1, 16 x 2304 19.8 / 18.7), but fewer of them where CTAs that add weights
  // wait behind them (16 x 1152 with weights: by the first rule 17.5, by the second 16.0).
  const int64_t per_row = a.first == nullptr
                              ? a.parts
                              : std::min((a.max_ctx + a.partition - 1) / a.partition,
                                         a.workers / (a.batch * a.hkv) + 1);
  int wpr = per_row >= 128 ? 32 : per_row >= 32 ? 8 : 1;
  const int64_t chunk = a.scores == nullptr ? 4 : 8, most = a.scores == nullptr ? 2048 : 1024;
  while (wpr < 8 && per_row > chunk * wpr && 2 * rows * wpr <= most) wpr *= 2;
  const int64_t merge = wpr == 32 ? rows : (rows * wpr + 7) / 8;
  // CTAs that add: one per 1024 tokens of a pair, but no more than about six per SM,
  // each then walking on: finding M and L costs a CTA as much as the tokens of one
  // such step (64 ragged sequences of up to 8192 tokens, 8 kv heads of 4 query heads,
  // fp16 / 4-bit decode with weights, us: 263 / 117; one step per CTA 265 / 122).
  const int64_t pairs = a.batch * a.hkv;
  int64_t chunks = 0;
  if (a.scores != nullptr) {
    chunks = std::max<int64_t>(1, (a.max_ctx + kAddTokens - 1) / kAddTokens);
    chunks = std::min(chunks, std::max<int64_t>(1, 6 * int64_t(ctx.sm_count) / pairs));
  }
  if (merge + pairs * chunks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  p.merge_blocks = static_cast<int>(merge);
  p.add_chunks = static_cast<int>(chunks);
  const unsigned grid = static_cast<unsigned>(merge + pairs * chunks);
  return a.d == 64 ? by_warps<64>(p, grid, wpr, a.bf16, ctx.stream)
                   : by_warps<128>(p, grid, wpr, a.bf16, ctx.stream);
}

}  // namespace fab
