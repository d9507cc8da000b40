// Eviction of cached tokens by their accumulated attention weights: per (sequence,
// kv head) the tokens to keep (the first `sinks`, the last `recent`, the largest
// totals of the rest, ties to the lower index), then their rows moved, in order,
// into the sequence's new pages.
#include <algorithm>

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
  FastDiv by_bs;
  int vector;  // four tokens from a multiple of four are one aligned load
};

constexpr int kBins = 2048;
// CTAs of a cluster. 16 (beyond the portable size) ran one cluster after another:
// 8 heads of 131072 tokens took 499 us against 33 us with 8.
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

// Sum of v over the lanes before this one.
__device__ __forceinline__ int before_of(int v, int lane) {
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  return incl - v;
}

// One cluster per (sequence, kv head); CTA r of it has the r-th share of the
// candidates. The need-th largest key comes by a radix select, 11, 11 and 10 bits
// at a time: every CTA counts its keys, adds up the cluster's counts and finds the
// same bin. Then every warp counts its run of keys above and at that key, and,
// knowing the counts before it, writes the indices that stay in order. Keys go four
// at a time, the totals of four tokens being one load where pages allow it.
//
// A pass over few long sequences is bound by one SM's latency, hence the cluster;
// keys wait in shared memory between the passes (HELD). Loops stay rolled: the
// kernel is short, and with its passes unrolled it waited for instructions half the
// time (B200, 64 sequences of 4096 tokens, 8 heads: 42 us).
template <int T, bool HELD>
__global__ void __launch_bounds__(T) evict_select_kernel(const SelectParams p) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ int hist[2][kBins];
  __shared__ int coarse[2][kBins / 32];
  __shared__ int warp_gt[T / 32], warp_eq[T / 32];
  __shared__ int share_gt, share_eq;
  __shared__ uint32_t s_digit;
  __shared__ int s_left;
  __shared__ bool s_whole;
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
    // Unsigned: keep may be 2^31 - 1, past which j goes once more.
    for (unsigned int j = at; j < static_cast<unsigned int>(p.keep); j += step)
      kept[j] = j < static_cast<unsigned int>(len) ? static_cast<int>(j) : -1;
    return;
  }
  const int first = p.sinks, last = len - p.recent;  // candidates [first, last)
  for (int j = at; j < p.sinks; j += step) kept[j] = j;
  for (int j = at; j < p.recent; j += step) kept[p.keep - p.recent + j] = last + j;
  const int need = p.keep - p.sinks - p.recent;
  if (need == 0) return;
  const int* bt = p.bt + static_cast<size_t>(b) * p.max_blocks;
  // The tokens [0, last) in runs, one per warp, of whole 128, four tokens a lane.
  const int runs = ranks * (T / 32);
  const int per_warp = ((last + runs - 1) / runs + 127) / 128 * 128;
  const int share = per_warp * (T / 32);
  const long long begin = static_cast<long long>(rank) * share;
  const int mine = static_cast<int>(min(max(last - begin, 0ll), static_cast<long long>(share)));
  // Keys of tokens begin + j .. + 3; 0, below every key, where they are no candidates.
  auto global_keys = [&](int j) -> uint4 {
    const uint32_t i = static_cast<uint32_t>(begin + j);
    uint32_t k[4];
    if (p.vector) {
      const uint32_t in = p.by_bs.quotient(i);
      const int page = bt[in];
      float4 w = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (static_cast<unsigned>(page) < static_cast<unsigned>(p.num_blocks))
        w = *reinterpret_cast<const float4*>(
            p.weights + (static_cast<size_t>(page) * p.hkv + kvh) * p.bs + (i - in * p.bs));
      else
        report_status(p.status, 2u /* ATTN_DEVICE_BAD_BLOCK */, kSiteSelectBlock);
      k[0] = key_of(w.x);
      k[1] = key_of(w.y);
      k[2] = key_of(w.z);
      k[3] = key_of(w.w);
    } else {
#pragma unroll 1
      for (int u = 0; u < 4; ++u) {
        float w = -INFINITY;
        if (j + u < mine) {
          const uint32_t in = p.by_bs.quotient(i + u);
          const int page = bt[in];
          if (static_cast<unsigned>(page) < static_cast<unsigned>(p.num_blocks))
            w = p.weights[(static_cast<size_t>(page) * p.hkv + kvh) * p.bs + (i + u - in * p.bs)];
          else
            report_status(p.status, 2u /* ATTN_DEVICE_BAD_BLOCK */, kSiteSelectBlock);
        }
        k[3] = u == 3 ? key_of(w) : k[3];
        k[2] = u == 2 ? key_of(w) : k[2];
        k[1] = u == 1 ? key_of(w) : k[1];
        k[0] = u == 0 ? key_of(w) : k[0];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (begin + j + u < first || j + u >= mine) k[u] = 0u;
    return make_uint4(k[0], k[1], k[2], k[3]);
  };
#pragma unroll 1
  for (int j = tid; j < kBins; j += T) hist[0][j] = 0;
  if constexpr (HELD) {
#pragma unroll 2
    for (int j = 4 * tid; j < mine; j += 4 * T)
      *reinterpret_cast<uint4*>(keys + j) = global_keys(j);
  }
  auto four = [&](int j) -> uint4 {
    if constexpr (HELD) return *reinterpret_cast<const uint4*>(keys + j);
    return global_keys(j);
  };
  __syncthreads();

  uint32_t prefix = 0, mask = 0;
  int left = need;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digits = pass == 2 ? 1023u : 2047u;
    int* h = hist[pass & 1];
#pragma unroll 1
    for (int j = 4 * tid; j < mine; j += 4 * T) {
      const uint4 k = four(j);
      if (k.x != 0u && (k.x & mask) == prefix) atomicAdd(&h[(k.x >> shift) & digits], 1);
      if (k.y != 0u && (k.y & mask) == prefix) atomicAdd(&h[(k.y >> shift) & digits], 1);
      if (k.z != 0u && (k.z & mask) == prefix) atomicAdd(&h[(k.z >> shift) & digits], 1);
      if (k.w != 0u && (k.w & mask) == prefix) atomicAdd(&h[(k.w >> shift) & digits], 1);
    }
    __syncthreads();
    // Sums of 32 bins each. The cluster's counts are looked up in two steps, of these
    // sums and then of the 32 bins in question: reading all bins of the other CTAs
    // took 9500 cycles a pass, half of the kernel.
#pragma unroll 1
    for (int c = warp; c < kBins / 32; c += T / 32) {
      const int sum = __reduce_add_sync(0xffffffffu, h[32 * c + lane]);
      if (lane == 0) coarse[pass & 1][c] = sum;
    }
    cluster.sync();
    // The other buffer is counted into in the next pass; no CTA reads it any more
    // (all have passed the cluster barrier above).
#pragma unroll 1
    for (int j = tid; j < kBins; j += T) hist[(pass & 1) ^ 1][j] = 0;
    if (warp == 0) {
      // From the top, the sum and then the bin where the running count reaches `left`.
      int c0 = 0, c1 = 0, one = 0;
      const int top = kBins / 32 - 1 - 2 * lane;  // lane's sums: top, top - 1
#pragma unroll 4
      for (int r = 0; r < ranks; ++r) {
        const int* other = cluster.map_shared_rank(&coarse[pass & 1][0], r);
        c0 += other[top];
        c1 += other[top - 1];
      }
      int above = before_of(c0 + c1, lane);
      const bool first_sum = above < left && left <= above + c0;
      const bool second_sum = above + c0 < left && left <= above + c0 + c1;
      const unsigned found = __ballot_sync(0xffffffffu, first_sum || second_sum);
      const int from = __ffs(found) - 1;
      const int block = __shfl_sync(0xffffffffu, first_sum ? top : top - 1, from);
      int rest = __shfl_sync(0xffffffffu, left - above - (first_sum ? 0 : c0), from);
#pragma unroll 4
      for (int r = 0; r < ranks; ++r)
        one += cluster.map_shared_rank(h, r)[32 * block + 31 - lane];
      above = before_of(one, lane);
      if (above < rest && rest <= above + one) {
        s_digit = static_cast<uint32_t>(32 * block + 31 - lane);
        s_left = rest - above;
        s_whole = rest - above == one;
      }
    }
    __syncthreads();
    prefix |= s_digit << shift;
    left = s_left;
    mask |= digits << shift;
    if (s_whole) {
      // The whole bin stays (of distinct totals a bin of the second pass mostly holds
      // one): all above the key before its first, and the passes are over.
      prefix -= 1u;
      left = 0;
      break;
    }
  }

  // Above the key: all; at it: the first `left` of the candidates.
  int gt = 0, eq = 0;
  const int w0 = warp * per_warp, w1 = min(mine, w0 + per_warp);
#pragma unroll 1
  for (int j = w0 + 4 * lane; j < w1; j += 128) {
    const uint4 k = four(j);
    gt += (k.x > prefix) + (k.y > prefix) + (k.z > prefix) + (k.w > prefix);
    eq += (k.x == prefix) + (k.y == prefix) + (k.z == prefix) + (k.w == prefix);
  }
  gt = __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  if (lane == 0) {
    warp_gt[warp] = gt;
    warp_eq[warp] = eq;
  }
  __syncthreads();
  int g = lane < T / 32 ? warp_gt[lane] : 0, e = lane < T / 32 ? warp_eq[lane] : 0;
  if (warp == 0) {
    const int all_g = __reduce_add_sync(0xffffffffu, g), all_e = __reduce_add_sync(0xffffffffu, e);
    if (lane == 0) {
      share_gt = all_g;
      share_eq = all_e;
    }
  }
  cluster.sync();
  // Before this warp's run: its CTA's warps before it, and the CTAs before that.
  if (lane >= warp) g = e = 0;
  if (lane < rank) {
    g += *cluster.map_shared_rank(&share_gt, lane);
    e += *cluster.map_shared_rank(&share_eq, lane);
  }
  g = __reduce_add_sync(0xffffffffu, g);
  e = __reduce_add_sync(0xffffffffu, e);
#pragma unroll 1
  for (int j0 = w0; j0 < w1; j0 += 128) {
    const int j = j0 + 4 * lane;
    const uint4 k4 = j < w1 ? four(j) : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
    // Counts of this lane, above in the low half and at the key in the high one, and
    // their sums over the lanes before it.
    int mine2 = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) mine2 += (k[u] > prefix) + ((k[u] == prefix) << 16);
    int incl = mine2;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const int before = incl - mine2, all = __shfl_sync(0xffffffffu, incl, 31);
    int my_g = g + (before & 0xffff), my_e = e + (before >> 16);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool is_gt = k[u] > prefix, is_eq = k[u] == prefix;
      if (is_gt || (is_eq && my_e < left))
        kept[p.sinks + my_g + min(my_e, left)] = static_cast<int>(begin + j + u);
      my_g += is_gt;
      my_e += is_eq;
    }
    g += all & 0xffff;
    e += all >> 16;
  }
  // Shared memory stays until the others have read it.
  if (ranks > 1) cluster.sync();
}

// --------------------------------------------------------------------- move

struct MoveParams {
  uint8_t* arrays[kMaxEvictArrays];  // [num_blocks, hkv, bs, row bytes]
  int row_vecs[kMaxEvictArrays];     // row bytes / 16, 8, 4, 2 or 1
  FastDiv by_row[kMaxEvictArrays];
  int num_arrays;
  float* weights;
  const int* kept;
  const int* new_lens;
  const int* bt;
  const int* new_bt;
  DeviceStatus* status;
  int hkv, bs, num_blocks, max_blocks, new_max_blocks, keep;
  FastDiv by_bs;
};

constexpr int kMoveRows = 64;

// 64 rows of one (sequence, kv head) at a time. Four pieces a thread are read before
// they are written: a load does not pass a store that could be to the same address.
template <typename V>
__global__ void __launch_bounds__(256) evict_move_kernel(const MoveParams p) {
  constexpr int U = 4;
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
        const int in = p.by_bs.quotient(i), out = p.by_bs.quotient(j);
        const int src = p.bt[static_cast<size_t>(b) * p.max_blocks + in];
        const int dst = p.new_bt[static_cast<size_t>(b) * p.new_max_blocks + out];
        if (src < 0 || src >= p.num_blocks || dst < 0 || dst >= p.num_blocks) {
          report_status(p.status, 2u /* ATTN_DEVICE_BAD_BLOCK */, kSiteMoveBlock);
        } else {
          f = (static_cast<long long>(src) * p.hkv + kvh) * p.bs + (i - in * p.bs);
          t = (static_cast<long long>(dst) * p.hkv + kvh) * p.bs + (j - out * p.bs);
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
      for (int x0 = threadIdx.x; x0 < kMoveRows * rv; x0 += U * 256) {
        V v[U];
        long long at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int x = x0 + u * 256;
          at[u] = -1;
          if (x < kMoveRows * rv) {
            const int r = p.by_row[a].quotient(x), c = x - r * rv;
            if (from[r] >= 0) {
              v[u] = base[from[r] * rv + c];
              at[u] = to[r] * rv + c;
            }
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (at[u] >= 0) base[at[u]] = v[u];
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

template <int T, bool HELD>
cudaError_t launch_select(const SelectParams& s, unsigned pairs, int ranks, const LaunchCtx& ctx) {
  // Room for a share rounded up to whole runs of 128 keys per warp.
  const int64_t share = (static_cast<int64_t>(s.max_ctx) + ranks - 1) / ranks;
  const int64_t keys = HELD ? (share + 4 * T - 1) / (4 * T) * (4 * T) : 0;
  static SmemLimit limit;
  cudaError_t e = allow_smem(evict_select_kernel<T, HELD>, kMaxKeys * 4, limit);
  if (e != cudaSuccess) return e;
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
  return cudaLaunchKernelEx(&cfg, evict_select_kernel<T, HELD>, s);
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
  s.vector = a.bs % 4 == 0 && reinterpret_cast<uintptr_t>(a.weights) % 16 == 0 ? 1 : 0;
  const unsigned pairs = static_cast<unsigned>(a.batch * a.hkv);
  // CTAs per (sequence, kv head): as many as keep the SMs busy, of 2048 tokens at
  // least; small CTAs (several per SM) where a share is small.
  int ranks = 1;
  while (ranks < kMaxCluster && static_cast<int64_t>(pairs) * ranks * 2 <= ctx.sm_count &&
         a.max_ctx / (ranks * 2) >= 2048)
    ranks *= 2;
  const int64_t share = (a.max_ctx + ranks - 1) / ranks;
  cudaError_t e = share > kMaxKeys ? launch_select<1024, false>(s, pairs, ranks, ctx)
                  : share > 8192   ? launch_select<1024, true>(s, pairs, ranks, ctx)
                                   : launch_select<256, true>(s, pairs, ranks, ctx);
  const int64_t most = std::min(a.keep, a.max_ctx);
  if (e != cudaSuccess || most == 0) return e;
  MoveParams m;
  int64_t vec = 16;
  for (int i = 0; i < a.num_arrays; ++i) {
    while (a.row_bytes[i] % vec != 0 || reinterpret_cast<uintptr_t>(a.arrays[i]) % vec != 0) vec /= 2;
    m.arrays[i] = static_cast<uint8_t*>(a.arrays[i]);
  }
  for (int i = 0; i < a.num_arrays; ++i) {
    m.row_vecs[i] = static_cast<int>(a.row_bytes[i] / vec);
    m.by_row[i] = FastDiv(m.row_vecs[i]);
  }
  m.by_bs = s.by_bs;
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
