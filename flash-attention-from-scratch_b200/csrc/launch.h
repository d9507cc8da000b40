// Host-side launchers of the kernels, called by the C ABI in api.cu. Each
// returns cudaSuccess or the launch error; argument checking is done by the
// caller.
#pragma once

#include <cstddef>
#include <cstdint>
#include <mutex>
#include <string>

#include <cuda_runtime.h>

#include "common.cuh"

namespace fab {

struct LaunchCtx {
  cudaStream_t stream;
  DeviceStatus* status;          // device status word of the current device
  unsigned long long timeout_ns; // limit of every bounded wait
  int sm_count;                  // SMs of the current device
};

// Allow a kernel `bytes` of dynamic shared memory on the current device, once per
// device (a function's attributes belong to the device that is current). `done` is
// the kernel's own, static.
struct SmemLimit {
  std::mutex mu;
  bool done[64] = {};
};
template <typename Kernel>
cudaError_t allow_smem(Kernel kernel, int bytes, SmemLimit& limit) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(limit.mu);
  if (limit.done[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  limit.done[dev] = e == cudaSuccess;
  return e;
}

// tcgen05 FlashAttention forward; q, k, v, o fp16 [bh, n, d], d in {64, 128}.
cudaError_t launch_flash_tc(const void* q, const void* k, const void* v, void* o, int64_t bh,
                            int64_t n, int d, bool causal, float scale, const LaunchCtx& ctx,
                            std::string* err);

// CUDA-core tiled online-softmax attention, same layout.
cudaError_t launch_flash_simt(const void* q, const void* k, const void* v, void* o, int64_t bh,
                              int64_t n, int d, bool causal, float scale, const LaunchCtx& ctx);

// Three-kernel attention with fp32 scores in `scores` ([bh, n, n]).
cudaError_t launch_naive(const void* q, const void* k, const void* v, void* o, float* scores,
                         int64_t bh, int64_t n, int d, bool causal, float scale,
                         const LaunchCtx& ctx);

struct DecodeArgs {
  const void* q;          // fp16 [batch, hq, d]
  const void* k_cache;    // fp16 [num_blocks, hkv, bs, d]
  const void* v_cache;
  const int32_t* block_tables;  // [batch, max_blocks]
  const int32_t* context_lens;  // [batch]
  void* out;              // fp16 [batch, hq, d]           (final mode)
  float* o_final;         // fp32 [batch, hq, d] partials   (partials mode)
  float* m_final;         // fp32 [batch, hq]
  float* l_final;
  int64_t batch, hq, hkv, d, bs, num_blocks, max_blocks, max_ctx, partition;
  float scale;
  void* workspace;
  size_t workspace_bytes;
  float* weights = nullptr;  // fp32 [num_blocks, hkv, bs]: attention weights are added (final mode)
};

// Workspace layout of the decode path.
size_t decode_workspace_bytes(int64_t batch, int64_t hq, int64_t d, int64_t max_ctx,
                              int64_t partition);

// The same with room for the scores behind it, for a call with weights.
size_t decode_weights_workspace_bytes(int64_t batch, int64_t hq, int64_t hkv, int64_t d,
                                      int64_t max_ctx, int64_t partition);

cudaError_t launch_paged_decode(const DecodeArgs& a, bool partials_mode, const LaunchCtx& ctx);

cudaError_t launch_merge(const float* o_parts, const float* m_parts, const float* l_parts,
                         int64_t num_parts, int64_t rows, int64_t d, int64_t o_part_stride,
                         int64_t ml_part_stride, void* out, const LaunchCtx& ctx);

// Query heads a token's scores are stored for (the group, rounded up to a power
// of two), and the bytes of fp32 scores [batch, hkv, max_ctx, score_heads].
int64_t score_heads(int64_t group);
size_t score_bytes(int64_t batch, int64_t hkv, int64_t group, int64_t max_ctx);

// The end of a decode launch in one kernel (csrc/finish.cu): fp32 parts merged
// into 16-bit rows, and, with scores, the attention weights added to the totals.
struct FinishArgs {
  const float* o;             // parts
  const float* m;
  const float* l;
  const int32_t* context_lens;
  // Where the parts are. first == null: of (sequence, query head) row r the parts
  // r * parts + s, s < ceil(length / partition). Else: equal runs of `workers` (or one
  // per stage, if that is fewer) over the stages of `partition` tokens, the part of
  // worker i and (sequence, kv head) pair j in slot i + j ([slots, group]); a pair in
  // one run has its rows written.
  const int32_t* first;       // [batch + 1] stages of one head before each sequence
  int64_t workers, partition, parts;
  const float* scores;        // [batch, hkv, max_ctx, score_heads] or null
  float* weights;             // [num_blocks, hkv, bs]
  const int32_t* block_tables;
  void* out;                  // fp16 (or bf16) [batch, hq, d]
  bool bf16;
  int64_t batch, hq, hkv, d, bs, num_blocks, max_blocks, max_ctx;
};
cudaError_t launch_finish(const FinishArgs& a, const LaunchCtx& ctx);

// ------------------------------------------------------------ 4-bit paged cache

struct Kv4CopyArgs {
  void* k;              // fp16 or bf16 [tokens, hkv, d]: read (append) or written, dense (read)
  void* v;
  bool bf16;
  int64_t token_stride[2], head_stride[2];  // of k and v, in elements (append)
  void* k_cache;        // uint8 [num_blocks, hkv, bs, row bytes]
  void* v_cache;
  const int64_t* slots; // [tokens]
  float* weights;       // append: [num_blocks, hkv, bs] to clear in the written slots, or null
  int64_t tokens, hkv, d, bs, num_blocks;
};
cudaError_t launch_kv4_append(const Kv4CopyArgs& a, const LaunchCtx& ctx);
cudaError_t launch_kv4_read(const Kv4CopyArgs& a, const LaunchCtx& ctx);

struct Kv4DecodeArgs {
  const void* q;        // fp16 or bf16 [batch, hq, d]
  bool bf16;
  const void* k_cache;  // uint8 [num_blocks, hkv, bs, row bytes]
  const void* v_cache;
  const int32_t* block_tables;
  const int32_t* context_lens;
  void* out;            // q's type [batch, hq, d]
  float* weights;       // fp32 [num_blocks, hkv, bs] or null
  int64_t batch, hq, hkv, d, bs, num_blocks, max_blocks, max_ctx;
  float scale;
  void* workspace;
  size_t workspace_bytes;
};
size_t kv4_decode_workspace_bytes(int64_t batch, int64_t hq, int64_t hkv, int64_t d, int64_t max_ctx,
                                  bool weights);
cudaError_t launch_kv4_decode(const Kv4DecodeArgs& a, const LaunchCtx& ctx);

// --------------------------------------------------------------------- eviction

// Most cache arrays one eviction moves.
constexpr int kMaxEvictArrays = 8;

struct EvictArgs {
  void* arrays[kMaxEvictArrays];  // [num_blocks, hkv, bs, row_bytes[i]]
  int64_t row_bytes[kMaxEvictArrays];
  int num_arrays;
  float* weights;                 // [num_blocks, hkv, bs]
  const int32_t* block_tables;    // [batch, max_blocks]
  const int32_t* context_lens;    // [batch]
  const int32_t* new_block_tables;  // [batch, new_max_blocks]
  int32_t* new_lens;              // [batch]
  int32_t* kept;                  // [batch, hkv, keep]
  int64_t batch, hkv, bs, num_blocks, max_blocks, max_ctx, new_max_blocks, keep, recent, sinks;
};
cudaError_t launch_evict(const EvictArgs& a, const LaunchCtx& ctx);

cudaError_t launch_selftest_wait(unsigned long long timeout_ns, const LaunchCtx& ctx);

// The prefill softmax's exponentials on n inputs: FMA-pipe polynomial, MUFU
// ex2.approx and exp2f (fp32 device arrays of n elements each).
cudaError_t launch_selftest_exp2(const float* x, float* y_poly, float* y_mufu, float* y_lib,
                                int64_t n, const LaunchCtx& ctx);

// Most ranks attn_exchange_merge_partials takes.
constexpr int kMaxPeers = 16;

// Context-parallel partials pushed to every peer over peer memory, then merged
// (csrc/exchange.cu). slots[q] / flags[q]: rank q's receive area for this call
// and its flag words, as device pointers valid on the current device.
cudaError_t launch_exchange_merge(float* const* slots, unsigned int* const* flags, int world,
                                  int rank, unsigned int epoch, int64_t rows, int d,
                                  int64_t slot_stride, void* out, const LaunchCtx& ctx);

// Size of the fixed device array that attn_paged_decode_noalloc uses as its
// split-K scratch (32 MiB per device that loads the library).
constexpr size_t kDecodeStaticScratchBytes = size_t(32) << 20;

// paged_decode (final fp16 output) with the scratch in that fixed array; the
// first call on a device looks up the array's device address. Fails with *err
// set when the problem needs more scratch than the array holds.
cudaError_t paged_decode_static_scratch(DecodeArgs a, const LaunchCtx& ctx, std::string* err);

}  // namespace fab
