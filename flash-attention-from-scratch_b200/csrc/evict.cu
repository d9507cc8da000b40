// Eviction of cached tokens by their accumulated attention weights: per (sequence, kv head) the tokens to keep (the first `sinks`, the last
// `recent`, the largest totals of the rest, ties to the lower index), then their
// rows moved, in order, into the sequence's new pages.
#include <algorithm>

#include "common.cuh"
#include "launch.h"

namespace fab {
namespace {

enum : unsigned int { kSiteSelectBlock = 231, kSiteMoveBlock = 232 };

// ------------------------------------------------------------------- select

struct SelectParams {
  const float* weights;
  const int* bt;
  const int* ctx;
  int* new_lens;  // [batch]
  int* kept;      // [batch, hkv, keep]
  DeviceStatus* status;
  int hkv, bs, num_blocks, max_blocks, max_ctx, keep, recent, sinks;
};

constexpr int kSelThreads = 1024;

// The totals as whole numbers in their order: NaN as the lowest total, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (w != w) w = -INFINITY;
  if (w == 0.f) w = 0.f;
  const uint32_t u = __float_as_uint(w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const SelectParams p) {
  __shared__ int hist[256];
  __shared__ int warp_gt[32], warp_eq[32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left;
  const int kvh = blockIdx.x % p.hkv, b = blockIdx.x / p.hkv;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int len = min(max(p.ctx[b], 0), p.max_ctx);
  int* kept = p.kept + static_cast<size_t>(blockIdx.x) * p.keep;
  if (kvh == 0 && tid == 0) p.new_lens[b] = min(len, p.keep);
  if (len <= p.keep) {
    for (int j = tid; j < p.keep; j += kSelThreads) kept[j] = j < len ? j : -1;
    return;
  }
  const int first = p.sinks, last = len - p.recent;  // candidates [first, last)
  for (int j = tid; j < p.sinks; j += kSelThreads) kept[j] = j;
  for (int j = tid; j < p.recent; j += kSelThreads) kept[p.keep - p.recent + j] = last + j;
  const int need = p.keep - p.sinks - p.recent;
  if (need == 0) return;
  const int* bt = p.bt + static_cast<size_t>(b) * p.max_blocks;
  auto key_at = [&](int i) -> uint32_t {
    const int page = bt[i / p.bs];
    if (page < 0 || page >= p.num_blocks) {
      report_status(p.status, 2u, kSiteSelectBlock);
      return 0u;
    }
    return key_of(p.weights[(static_cast<size_t>(page) * p.hkv + kvh) * p.bs + i % p.bs]);
  };
  // The need-th largest key, eight bits at a time.
  uint32_t prefix = 0, mask = 0;
  int left = need;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = first + tid; i < last; i += kSelThreads) {
      const uint32_t k = key_at(i);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1);
    }
    __syncthreads();
    if (warp == 0) {
      // Lane i sums bins 255 - 8 i .. 248 - 8 i; the bin where the running count
      // from the top reaches `left` holds the key.
      int c[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += c[j] = hist[255 - 8 * lane - j];
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      int above = incl - sum;
      if (above < left && left <= incl) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (above < left && left <= above + c[j]) {
            s_prefix = prefix | (static_cast<uint32_t>(255 - 8 * lane - j) << shift);
            s_left = left - above;
          }
          above += c[j];
        }
      }
    }
    __syncthreads();
    prefix = s_prefix;
    left = s_left;
    mask |= 255u << shift;
  }
  // Above the key: all; at it: the first `left`.
  int gt_base = 0, eq_base = 0;
  for (int i0 = first; i0 < last; i0 += kSelThreads) {
    const int i = i0 + tid;
    const uint32_t k = i < last ? key_at(i) : 0u;
    const bool gt = i < last && k > prefix, eq = i < last && k == prefix;
    const unsigned bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) {
      warp_gt[warp] = __popc(bg);
      warp_eq[warp] = __popc(be);
    }
    __syncthreads();
    int g = gt_base, e = eq_base, g_all = 0, e_all = 0;
    for (int w = 0; w < kSelThreads / 32; ++w) {
      if (w < warp) {
        g += warp_gt[w];
        e += warp_eq[w];
      }
      g_all += warp_gt[w];
      e_all += warp_eq[w];
    }
    const unsigned below = (1u << lane) - 1u;
    g += __popc(bg & below);
    e += __popc(be & below);
    if (gt || (eq && e < left)) kept[p.sinks + g + min(e, left)] = i;
    gt_base += g_all;
    eq_base += e_all;
    __syncthreads();
  }
}

// --------------------------------------------------------------------- move

struct MoveParams {
  uint8_t* arrays[kMaxEvictArrays];  // [num_blocks, hkv, bs, row bytes]
  int row_vecs[kMaxEvictArrays];     // row bytes / 16, 8, 4, 2 or 1
  int num_arrays;
  float* weights;
  const int* kept;
  const int* new_lens;
  const int* bt;
  const int* new_bt;
  DeviceStatus* status;
  int hkv, bs, num_blocks, max_blocks, new_max_blocks, keep;
};

constexpr int kMoveRows = 64;

template <typename V>
__global__ void __launch_bounds__(256) evict_move_kernel(const MoveParams p) {
  __shared__ long long from[kMoveRows], to[kMoveRows];  // row numbers; from < 0: not moved
  const int kvh = blockIdx.x % p.hkv, b = blockIdx.x / p.hkv;
  const int n = p.new_lens[b];
  for (long long j0 = static_cast<long long>(blockIdx.y) * kMoveRows; j0 < n;
       j0 += static_cast<long long>(gridDim.y) * kMoveRows) {
  __syncthreads();
  if (threadIdx.x < kMoveRows) {
    const int j = static_cast<int>(j0) + threadIdx.x;
    long long f = -1, t = 0;
    if (j < n) {
      const int i = p.kept[static_cast<size_t>(blockIdx.x) * p.keep + j];
      const int src = p.bt[static_cast<size_t>(b) * p.max_blocks + i / p.bs];
      const int dst = p.new_bt[static_cast<size_t>(b) * p.new_max_blocks + j / p.bs];
      if (src < 0 || src >= p.num_blocks || dst < 0 || dst >= p.num_blocks) {
        report_status(p.status, 2u, kSiteMoveBlock);
      } else {
        f = (static_cast<long long>(src) * p.hkv + kvh) * p.bs + i % p.bs;
        t = (static_cast<long long>(dst) * p.hkv + kvh) * p.bs + j % p.bs;
        if (f == t) f = -1;
      }
    }
    from[threadIdx.x] = f;
    to[threadIdx.x] = t;
    if (f >= 0) p.weights[t] = p.weights[f];
  }
  __syncthreads();
  for (int a = 0; a < p.num_arrays; ++a) {
    const int rv = p.row_vecs[a];
    V* base = reinterpret_cast<V*>(p.arrays[a]);
    for (int x = threadIdx.x; x < kMoveRows * rv; x += 256) {
      const int r = x / rv, c = x - r * rv;
      if (from[r] >= 0) base[to[r] * rv + c] = base[from[r] * rv + c];
    }
  }
  }
}

// CTAs along y for `n` items, `per` at a time; a kernel walks on by the grid.
unsigned grid_y(int64_t n, int64_t per) {
  return static_cast<unsigned>(std::min<int64_t>((n + per - 1) / per, 65535));
}

}  // namespace

cudaError_t launch_evict(const EvictArgs& a, const LaunchCtx& ctx) {
  SelectParams s;
  s.weights = a.weights;
  s.bt = a.block_tables;
  s.ctx = a.context_lens;
  s.new_lens = a.new_lens;
  s.kept = a.kept;
  s.status = ctx.status;
  s.hkv = static_cast<int>(a.hkv);
  s.bs = static_cast<int>(a.bs);
  s.num_blocks = static_cast<int>(a.num_blocks);
  s.max_blocks = static_cast<int>(a.max_blocks);
  s.max_ctx = static_cast<int>(a.max_ctx);
  s.keep = static_cast<int>(a.keep);
  s.recent = static_cast<int>(a.recent);
  s.sinks = static_cast<int>(a.sinks);
  const unsigned pairs = static_cast<unsigned>(a.batch * a.hkv);
  evict_select_kernel<<<pairs, kSelThreads, 0, ctx.stream>>>(s);
  cudaError_t e = cudaGetLastError();
  const int64_t most = std::min(a.keep, a.max_ctx);
  if (e != cudaSuccess || most == 0) return e;
  MoveParams m;
  int64_t vec = 16;
  for (int i = 0; i < a.num_arrays; ++i) {
    while (a.row_bytes[i] % vec != 0 || reinterpret_cast<uintptr_t>(a.arrays[i]) % vec != 0) vec /= 2;
    m.arrays[i] = static_cast<uint8_t*>(a.arrays[i]);
  }
  for (int i = 0; i < a.num_arrays; ++i) m.row_vecs[i] = static_cast<int>(a.row_bytes[i] / vec);
  m.num_arrays = a.num_arrays;
  m.weights = a.weights;
  m.kept = a.kept;
  m.new_lens = a.new_lens;
  m.bt = a.block_tables;
  m.new_bt = a.new_block_tables;
  m.status = ctx.status;
  m.hkv = s.hkv;
  m.bs = s.bs;
  m.num_blocks = s.num_blocks;
  m.max_blocks = s.max_blocks;
  m.new_max_blocks = static_cast<int>(a.new_max_blocks);
  m.keep = s.keep;
  const dim3 grid(pairs, grid_y(most, kMoveRows));
  switch (vec) {
    case 16: evict_move_kernel<uint4><<<grid, 256, 0, ctx.stream>>>(m); break;
    case 8: evict_move_kernel<uint2><<<grid, 256, 0, ctx.stream>>>(m); break;
    case 4: evict_move_kernel<uint32_t><<<grid, 256, 0, ctx.stream>>>(m); break;
    case 2: evict_move_kernel<uint16_t><<<grid, 256, 0, ctx.stream>>>(m); break;
    default: evict_move_kernel<uint8_t><<<grid, 256, 0, ctx.stream>>>(m); break;
  }
  return cudaGetLastError();
}

}  // namespace fab
