// Eviction of cached tokens by their accumulated attention weights: per (sequence,
// kv head) the tokens to keep (the first `sinks`, the last `recent`, the largest
// totals of the rest, ties to the lower index), then their rows moved, in order,
// into the sequence's new pages.
#include <algorithm>
#include <mutex>

#include <cooperative_groups.h>

#include "kv4.cuh"
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
  int key_room;  // keys that fit into the launch's shared memory
  FastDiv by_bs;
};

constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
// Keys a CTA holds in shared memory; a longer share is read again in every pass.
constexpr int kMaxKeys = 48 * 1024;

// The totals as whole numbers in their order: NaN as the lowest total, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (w != w) w = -INFINITY;
  if (w == 0.f) w = 0.f;
  const uint32_t u = __float_as_uint(w);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// One cluster per (sequence, kv head); CTA r of it has the r-th share of the
// candidates. The need-th largest key comes by a radix select, 11, 11 and 10 bits
// at a time: every CTA counts its keys, adds up the cluster's counts and finds the
// same bin. Then every warp counts its run of keys above and at that key, and,
// knowing the counts before it, writes the indices that stay in order.
//
// A pass over few long sequences is bound by one SM's latency, hence the cluster;
// keys wait in shared memory between the passes.
template <int T>
__global__ void __launch_bounds__(T) evict_select_kernel(const SelectParams p) {
  namespace cg = cooperative_groups;
  extern __shared__ uint32_t keys[];
  __shared__ int hist[2][kBins];
  __shared__ int warp_sum_s[T / 32];
  __shared__ int warp_gt[T / 32], warp_eq[T / 32];
  __shared__ int share_gt, share_eq;
  __shared__ uint32_t s_digit;
  __shared__ int s_left;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int pair = blockIdx.x / ranks;
  const int kvh = pair % p.hkv, b = pair / p.hkv;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int len = min(max(p.ctx[b], 0), p.max_ctx);
  int* kept = p.kept + static_cast<size_t>(pair) * p.keep;
  const int at = rank * T + tid, step = ranks * T;
  if (kvh == 0 && at == 0) p.new_lens[b] = min(len, p.keep);
  if (len <= p.keep) {  // the whole cluster alike
    for (int j = at; j < p.keep; j += step) kept[j] = j < len ? j : -1;
    return;
  }
  const int first = p.sinks, last = len - p.recent;  // candidates [first, last)
  for (int j = at; j < p.sinks; j += step) kept[j] = j;
  for (int j = at; j < p.recent; j += step) kept[p.keep - p.recent + j] = last + j;
  const int need = p.keep - p.sinks - p.recent;
  if (need == 0) return;
  const int* bt = p.bt + static_cast<size_t>(b) * p.max_blocks;
  // A run of keys per warp, a multiple of 32, so that lanes and keys keep their order.
  const int per_warp = ((last - first + ranks * (T / 32) - 1) / (ranks * (T / 32)) + 31) / 32 * 32;
  const long long begin = first + static_cast<long long>(rank) * per_warp * (T / 32);
  const int share = per_warp * (T / 32);
  const int mine = static_cast<int>(min(max(last - begin, 0ll), static_cast<long long>(share)));
  auto global_key = [&](int j) -> uint32_t {
    const uint32_t i = static_cast<uint32_t>(begin + j), in = p.by_bs.quotient(i);
    const int page = bt[in];
    if (page < 0 || page >= p.num_blocks) {
      report_status(p.status, 2u /* ATTN_DEVICE_BAD_BLOCK */, kSiteSelectBlock);
      return 0u;
    }
    return key_of(p.weights[(static_cast<size_t>(page) * p.hkv + kvh) * p.bs + (i - in * p.bs)]);
  };
  const bool held = share <= p.key_room;
  for (int j = tid; j < kBins; j += T) hist[0][j] = 0;
  if (held) {
#pragma unroll 8
    for (int j = tid; j < mine; j += T) keys[j] = global_key(j);
  }
  __syncthreads();

  uint32_t prefix = 0, mask = 0;
  int left = need;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digits = pass == 2 ? 1023u : 2047u;
    int* h = hist[pass & 1];
    for (int j = tid; j < mine; j += T) {
      const uint32_t k = held ? keys[j] : global_key(j);
      if ((k & mask) == prefix) atomicAdd(&h[(k >> shift) & digits], 1);
    }
    cluster.sync();
    // Bins from the top, kBins / T a thread: the cluster's counts, and the bin where
    // the running count reaches `left`.
    constexpr int B = kBins / T;
    int c[B], sum = 0;
#pragma unroll
    for (int j = 0; j < B; ++j) {
      c[j] = 0;
      for (int r = 0; r < ranks; ++r)
        c[j] += cluster.map_shared_rank(h, r)[kBins - 1 - (tid * B + j)];
      sum += c[j];
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) warp_sum_s[warp] = incl;
    // The other buffer is counted into in the next pass; no CTA reads it any more
    // (all have passed the cluster barrier above).
    for (int j = tid; j < kBins; j += T) hist[(pass & 1) ^ 1][j] = 0;
    __syncthreads();
    int above = incl - sum;
#pragma unroll
    for (int w = 0; w < T / 32; ++w)
      if (w < warp) above += warp_sum_s[w];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      if (above < left && left <= above + c[j]) {
        s_digit = static_cast<uint32_t>(kBins - 1 - (tid * B + j));
        s_left = left - above;
      }
      above += c[j];
    }
    __syncthreads();
    prefix |= s_digit << shift;
    left = s_left;
    mask |= digits << shift;
  }

  // Above the key: all; at it: the first `left` of the candidates.
  int gt = 0, eq = 0;
  const int w0 = warp * per_warp, w1 = min(mine, w0 + per_warp);
  for (int j = w0 + lane; j < w1; j += 32) {
    const uint32_t k = held ? keys[j] : global_key(j);
    gt += k > prefix;
    eq += k == prefix;
  }
  gt = __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  if (lane == 0) {
    warp_gt[warp] = gt;
    warp_eq[warp] = eq;
  }
  __syncthreads();
  if (tid == 0) {
    int g = 0, e = 0;
    for (int w = 0; w < T / 32; ++w) {
      g += warp_gt[w];
      e += warp_eq[w];
    }
    share_gt = g;
    share_eq = e;
  }
  cluster.sync();
  int g = 0, e = 0;
  for (int r = 0; r < rank; ++r) {
    g += *cluster.map_shared_rank(&share_gt, r);
    e += *cluster.map_shared_rank(&share_eq, r);
  }
  for (int w = 0; w < warp; ++w) {
    g += warp_gt[w];
    e += warp_eq[w];
  }
  const unsigned below = (1u << lane) - 1u;
  for (int j0 = w0; j0 < w1; j0 += 32) {
    const int j = j0 + lane;
    const uint32_t k = j < w1 ? (held ? keys[j] : global_key(j)) : 0u;
    const bool is_gt = j < w1 && k > prefix, is_eq = j < w1 && k == prefix;
    const unsigned bg = __ballot_sync(0xffffffffu, is_gt), be = __ballot_sync(0xffffffffu, is_eq);
    const int my_g = g + __popc(bg & below), my_e = e + __popc(be & below);
    if (is_gt || (is_eq && my_e < left))
      kept[p.sinks + my_g + min(my_e, left)] = static_cast<int>(begin + j);
    g += __popc(bg);
    e += __popc(be);
  }
  // Shared memory stays until the others have read it.
  cluster.sync();
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

namespace {

template <int T>
cudaError_t launch_select(SelectParams s, unsigned pairs, int ranks, int64_t share,
                          const LaunchCtx& ctx) {
  // Room for a share rounded up to whole runs of 32 keys per warp.
  const int64_t keys = std::min<int64_t>((share + T - 1) / T * T, kMaxKeys);
  s.key_room = static_cast<int>(keys);
  // Per device: a function's attributes belong to the device that is current.
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!done[dev]) {
      e = cudaFuncSetAttribute(evict_select_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               kMaxKeys * 4);
      if (e != cudaSuccess) return e;
      done[dev] = true;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(pairs * static_cast<unsigned>(ranks));
  cfg.blockDim = dim3(T);
  cfg.dynamicSmemBytes = static_cast<size_t>(keys) * 4;
  cfg.stream = ctx.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, evict_select_kernel<T>, s);
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
  s.by_bs = FastDiv(a.bs);
  const unsigned pairs = static_cast<unsigned>(a.batch * a.hkv);
  // CTAs per (sequence, kv head): as many as keep the SMs busy, of 2048 tokens at
  // least; small CTAs (several per SM) where a share is small.
  int ranks = 1;
  while (ranks < kMaxCluster && static_cast<int64_t>(pairs) * ranks * 2 <= ctx.sm_count &&
         a.max_ctx / (ranks * 2) >= 2048)
    ranks *= 2;
  const int64_t share = (a.max_ctx + ranks - 1) / ranks;
  cudaError_t e = share > 8192 ? launch_select<1024>(s, pairs, ranks, share, ctx)
                               : launch_select<256>(s, pairs, ranks, share, ctx);
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
