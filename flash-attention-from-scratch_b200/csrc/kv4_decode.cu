// Decode attention of one query token per sequence over the 4-bit paged cache
// (row layout: kv4.cuh): scores in log2 units, a running maximum and sum, and
// fp32 (o, m, l) parts that the finish kernel (finish.cu) merges.
//
// A token costs 160 bytes of K and V per kv head at head_dim 128 where fp16 takes
// 512, so at the memory's rate an SM has about 7 cycles for a token: the kernel is
// laid out to spend few instructions on it.
//
//   * Warps are independent pipelines: bulk copies of whole page runs into a
//     per-warp ring of stages (48 tokens at head_dim 128, 64 at 64), signalled by
//     mbarriers.
//   * The stages of all (sequence, kv head) rows, in that order, are dealt out to
//     the resident warps in equal runs (Runs, kv4.cuh): of S stages a warp takes
//     S / n or one more, whatever the lengths are. A row that lies in one warp's run is
//     written at once; of the others each warp leaves a part, in slot i + row,
//     which no two (warp, row) pairs share, since along the runs one of the two
//     grows at each step: n + rows slots are enough for any lengths.
//     Where there are few short rows, a CTA has one, its warps share out the stages and
//     it merges their parts itself (JOIN): one launch instead of two.
//   * Both products run on the tensor cores (mma.sync m16n8k16) with the cached
//     rows as the 16-row operand A and the query heads of the kv head as the 8
//     columns of B, so up to 8 heads cost what one does:
//         S^T [16 tokens x 8 heads] = K [16 x D] q^T
//         O^T [16 columns x 8 heads] += V^T [16 x 16 tokens] P^T
//   * Codes reach the tensor cores without arithmetic. A 4-bit code n in bits 0-3
//     of an fp16 is the subnormal n 2^-24 (in bits 4-7: n 2^-20), which the tensor
//     cores multiply exactly; so one AND makes two operands, and the row layout
//     puts the codes that an operand register pairs 16 bits apart. q is halved four
//     times for the codes in bits 4-7; of O the odd columns are divided by 16 at
//     the end.
//   * A group's scale stays outside the product over the codes: K has one fp32
//     accumulator per group, combined as sum_w scale_w acc_w in fp32; V's scales
//     multiply P before each group's columns. The lows are one product more:
//     low . (sum of q over the group), with that sum as two fp16 terms (22 bits).
//   * The sums over a long context are kept centred. sum p v is near 0 where
//     sum p scale code and sum p low are not, so V is summed as
//         sum (p scale) (code - c) + sum p (low + c scale),   c = 8, 7 in turn:
//     one product with the constants -c per tile and group, added once a stage, and
//     fp16 middles in the lows' place. (Summing codes and lows as they are left outputs of 131072
//     tokens off by 0.8 %, from the tensor cores' rounding of the large sums alone.)
//     P is two fp16 terms, P scale one, rounded once from both: the one rounding of
//     a token's weight, like P's in fp16 attention.
//   * P is held times 2^up, up = 14 - floor(log2(max(1, S))) with S the largest scale of V
//     that the warp has met in the row: P scale stays below 2^15, and has fp16's 11 bits
//     down to P scale = 2^-28 max(1, S). With a fixed factor of 4 the small weights'
//     products with small scales were below fp16's range: for V of 1e-4, 32768 tokens and
//     scores of deviation 2 the RMS error at bf16 output was 4.3 to 5 times that of the
//     roundings named here. `up` only falls, once or twice a row, and the sums so far with
//     it, by the factor that makes them follow the running maximum. (64 x 8192 at head_dim
//     128: 96.7 -> 99.1 us, 8 x 131072: 261 -> 264; 64 x 8192 at 64: 64.7.)
//   * q of a head is scaled by the power of two that brings its largest value into
//     [2^7, 2^8), so that fp16 holds every bit that matters of an fp16 or bf16 q.
#include <algorithm>

#include "kv4.cuh"
#include "launch.h"

namespace fab {
namespace {

enum : unsigned int { kSiteKv4Wait = 221, kSiteKv4Drain = 222, kSiteKv4Block = 223 };

constexpr int kLaunchBatch = 2048;  // sequences per launch (their lengths live in shared memory)

// Flags of a stage beside its tokens (at most 64): the first and the last of its
// row for this warp, and, with the last, the row lies wholly in this warp's run.
enum : int { kTokens = 127, kFirst = 128, kLast = 256, kWhole = 512 };

template <int D>
struct Kv4Cfg {
  using R = Kv4Row<D>;
  // Warps per CTA (one CTA per SM) and tokens per stage. Measured at head_dim 128 (us,
  // 64 ragged sequences of up to 8192 tokens / 8 of 131072, 8 kv heads; one of 700):
  // 12 warps of 48 tokens 100 / 267, 8.9; 16 of 32 (128 registers, some spilled) 100 /
  // 268, 10.2; 8 of 64 106 / 292, 9.0. At 64 (64 x 8192, 64 query over 8 kv heads): 16
  // warps of 64 tokens 66, 12 70, 8 78. (Before the centring product was one per group,
  // the parts of few rows were merged by more warps and P was held by V's scales: the 12
  // of 48 are at 99 / 264, 8.2 with that, the 16 of 64 at 64.)
  static constexpr int W = D == 64 ? 16 : 12;
  static constexpr int THREADS = W * 32;
  static constexpr int NG = R::NG;
  static constexpr int ROW = R::BYTES;
  static constexpr int TOK = D == 64 ? 64 : 48;
  static constexpr int MT = TOK / 16;   // 16-token tiles of a stage
  static constexpr int KV = TOK * ROW;  // K (or V) bytes of one stage
  static constexpr int STAGE = 2 * KV;
  static constexpr int STAGES = 2;
  static constexpr int RING = STAGES * STAGE;
  static constexpr int ML_OFF = 8 * D * 4;  // JOIN: a part's m and l, behind its o, in the ring
  static_assert(ML_OFF + 8 * 8 <= RING, "a part in the ring");
  static constexpr int BAR_OFF = W * RING;
  static constexpr int META_OFF = (BAR_OFF + W * STAGES * 8 + 15) / 16 * 16;
  static constexpr int PREFIX_OFF = META_OFF + W * STAGES * 16;
  static constexpr int CTX_OFF = PREFIX_OFF + (kLaunchBatch + 1) * 4;
  static constexpr int CENTRE_OFF = (CTX_OFF + kLaunchBatch * 4 + 15) / 16 * 16;
  static constexpr int SMEM = CENTRE_OFF + 16 + 16;  // + the abort flag
  static_assert(STAGE % 16 == 0 && KV % 16 == 0 && BAR_OFF % 16 == 0, "bulk copy alignment");
  static_assert(SMEM <= 227 * 1024, "shared memory per CTA");
};

struct Kv4DecParams {
  const void* q;          // [batch, hq, D] fp16 or bf16
  const uint8_t* kc;      // [num_blocks, hkv, bs, row]
  const uint8_t* vc;
  const int* bt;
  const int* ctx;
  void* out;              // q's type [batch, hq, D]: rows that one warp has whole
  float* o_part;          // [slots, group, D]
  float* m_part;          // [slots, group]
  float* l_part;
  int* first;             // [batch + 1]: stages of one head before each sequence
  float* scores;          // SCORED: [batch, hkv, max_ctx, gp] log2-unit scores
  float* weights;         // SCORED and JOIN: [num_blocks, hkv, bs]
  FastDiv by_bs;
  DeviceStatus* status;
  unsigned long long timeout_ns;
  unsigned int block_stride;  // bytes between physical blocks
  int batch, hq, hkv, group, gp, bs, max_blocks, num_blocks, max_ctx;
  float scale_log2;
};

// D (16x8, fp32) += A (16x16, fp16, rows) B (16x8, fp16, columns).
__device__ __forceinline__ void mma_k16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// D = A B.
__device__ __forceinline__ void mma_k16_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                            uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// D = A B with A 16x8.
__device__ __forceinline__ void mma_k8_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5}, {%6}, "
      "{%7, %7, %7, %7};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}

// Transpose of an 8x8 fp16 matrix whose row i lanes 4 i .. 4 i + 3 hold in pairs.
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b),
                            *reinterpret_cast<__half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Pairs of fp16: 8 and 7; and what centres an even and an odd row of V (8 and 7 codes
// below, so that the middle of the codes is 0 on average), in the codes' unit 2^-24.
constexpr uint32_t kEight = 0x48004800u, kSeven = 0x47004700u, kCentre = 0x80078008u;

// N 32-bit words (1, 2 or 4) of shared memory in one load.
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&r)[N], const uint8_t* p) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    r[0] = v.x; r[1] = v.y;
  } else {
    r[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// 2^e as a float, -126 <= e <= 127.
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

// JOIN: a CTA has one (sequence, kv head) row, dealt out in equal runs to its warps,
// and merges their parts itself, in shared memory.
template <int D, typename T, bool SCORED, bool JOIN>
__global__ void __launch_bounds__(Kv4Cfg<D>::THREADS, 1) kv4_decode_kernel(const Kv4DecParams p) {
  using C = Kv4Cfg<D>;
  constexpr int NG = C::NG, ROW = C::ROW, CODES = C::R::CODES, kTok = C::TOK, MT = C::MT;
  extern __shared__ __align__(128) uint8_t smem[];
  // By a shuffle, which tells the compiler that it is the same in all lanes: the
  // producer's state then stays in uniform registers, which bulk copies are issued from.
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  const int g4 = lane >> 2, t4 = lane & 3;
  uint8_t* ring = smem + warp * C::RING;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF) + warp * C::STAGES;
  int4* meta = reinterpret_cast<int4*>(smem + C::META_OFF) + warp * C::STAGES;
  int* prefix = reinterpret_cast<int*>(smem + C::PREFIX_OFF);
  int* ctx_s = reinterpret_cast<int*>(smem + C::CTX_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::SMEM - 16);
  // The merge that follows may be scheduled now; it waits for this launch's end
  // before it reads the parts.
  if constexpr (!JOIN) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // Lengths and the stages of one head before each sequence, which the finish
  // kernel goes by too.
  const int my_b = static_cast<int>(blockIdx.x) / p.hkv;  // JOIN
  int my_len = 0;
  if constexpr (JOIN) {
    my_len = min(max(p.ctx[my_b], 0), p.max_ctx);
  } else {
    for (int b = threadIdx.x; b < p.batch; b += C::THREADS)
      ctx_s[b] = min(max(p.ctx[b], 0), p.max_ctx);
  }
  auto len_of = [&](int b) { return JOIN ? my_len : ctx_s[b]; };
  if (threadIdx.x < C::W * C::STAGES)
    mbar_init(reinterpret_cast<uint64_t*>(smem + C::BAR_OFF) + threadIdx.x, 1);
  if (threadIdx.x < 4)
    reinterpret_cast<uint32_t*>(smem + C::CENTRE_OFF)[threadIdx.x] = kCentre;
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if constexpr (!JOIN) {
    if (warp == 0) {
      const int per = (p.batch + 31) / 32;
      const int b0 = lane * per;
      int sum = 0;
      for (int i = 0; i < per; ++i)
        if (b0 + i < p.batch) sum += (ctx_s[b0 + i] + kTok - 1) / kTok;
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      int run = incl - sum;
      for (int i = 0; i < per; ++i) {
        if (b0 + i < p.batch) {
          prefix[b0 + i] = run;
          run += (ctx_s[b0 + i] + kTok - 1) / kTok;
        }
      }
      if (lane == 31) prefix[p.batch] = incl;
    }
    __syncthreads();
    if (blockIdx.x == 0) {
      for (int b = threadIdx.x; b <= p.batch; b += C::THREADS) p.first[b] = prefix[b];
    }
  }

  // This warp's run of stages. Warps next to each other in number are on different
  // SMs, so that a small call spreads over all of them.
  const unsigned int worker = JOIN ? warp : warp * gridDim.x + blockIdx.x;
  const Runs runs(JOIN ? (my_len + kTok - 1) / kTok
                       : static_cast<unsigned int>(prefix[p.batch]) * p.hkv,
                  JOIN ? C::W : C::W * gridDim.x);
  const unsigned int run0 = runs.begin(worker);
  unsigned int left = worker < runs.workers ? runs.begin(worker + 1) - run0 : 0u;

  // ---------------------------------------------------------- producer state
  int pb = 0, pkvh = 0, pst = 0, pnst = 0;  // the next stage: sequence, kv head, stage of that row
  int ppg = 0, poff = 0;                    // page of the row and token in it where it begins
  bool pfirst = true, pwhole = true;        // it is this warp's first of the row; from the row's first
  // K rows of the kv head in pages [bt_base, bt_base + 32) of the sequence, one page per
  // lane, and the block-table entries of the next 32, which are on their way meanwhile.
  int bt_base = 0, bt_next = 0;
  unsigned long long bt_rows = 0;
  const unsigned long long v_less_k =
      reinterpret_cast<unsigned long long>(p.vc) - reinterpret_cast<unsigned long long>(p.kc);
  bool fresh = false;  // the row's first window is still to be taken
  unsigned int p_slot = 0, c_slot = 0, c_parity = 0, ahead = 0;
  const bool leader = elect_one();

  auto table = [&](int pg) {
    return pg < p.max_blocks ? p.bt[static_cast<size_t>(pb) * p.max_blocks + pg] : 0;
  };
  // Takes the entries of bt_next, those of pages bt_base + lane, and asks for the next.
  auto window = [&]() {
    unsigned int page = static_cast<unsigned int>(bt_next);
    if (page >= static_cast<unsigned int>(p.num_blocks)) {  // never read outside the cache
      // An entry past the sequence's last page is not looked at.
      if ((bt_base + lane) * static_cast<long long>(p.bs) < len_of(pb))
        report_status(p.status, 2u /* ATTN_DEVICE_BAD_BLOCK */, kSiteKv4Block);
      page = 0;
    }
    bt_rows = reinterpret_cast<unsigned long long>(p.kc) +
              static_cast<unsigned long long>(page) * p.block_stride +
              static_cast<unsigned long long>(pkvh) * p.bs * ROW;
    bt_next = table(bt_base + 32 + lane);
  };
  auto open_row = [&]() {
    pfirst = true;
    pwhole = pst == 0;
    ppg = pst * kTok / p.bs;
    poff = pst * kTok - ppg * p.bs;
    bt_base = ppg;
    bt_next = table(bt_base + lane);
    fresh = true;
  };

  if constexpr (JOIN) {
    pb = my_b;
    pkvh = static_cast<int>(blockIdx.x) - my_b * p.hkv;
    pnst = (my_len + kTok - 1) / kTok;
    pst = static_cast<int>(run0);
    if (left > 0) open_row();
  } else if (left > 0) {
    int lo = 0, hi = p.batch - 1;  // last sequence whose first stage is <= run0
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (static_cast<unsigned int>(prefix[mid]) * p.hkv <= run0) lo = mid; else hi = mid - 1;
    }
    pb = lo;
    pnst = prefix[lo + 1] - prefix[lo];
    const unsigned int in_seq = run0 - static_cast<unsigned int>(prefix[lo]) * p.hkv;
    pkvh = static_cast<int>(in_seq / static_cast<unsigned int>(pnst));
    pst = static_cast<int>(in_seq) - pkvh * pnst;
    open_row();
  }

  // Issue the copies of the producer's next stage into its ring slot, page by page
  // from one elected lane, with operands that are the same in all lanes. (With a
  // page per lane the compiler puts a loop over the lanes around each copy.) Addresses
  // come 32 pages at a time, one per lane, and are handed out by shuffles.
  auto produce = [&]() {
    if (left == 0) return;
    uint8_t* dst = ring + p_slot * C::STAGE;
    uint64_t* bar = full + p_slot;
    const int t0 = pst * kTok;
    const int nt = min(kTok, len_of(pb) - t0);
    // Copies are of whole 16 bytes: where a row is not (40 bytes), an odd last token
    // brings the row after it along, which is in its page (the block size is even).
    int todo = ROW % 16 != 0 ? nt + (nt & 1) : nt;
    const bool row_end = pst + 1 == pnst;
    if (leader) {
      mbar_arrive_expect_tx(bar, 2 * todo * ROW);
      meta[p_slot] = make_int4(pb, pkvh, t0,
                               nt | (pfirst ? kFirst : 0) | (row_end || left == 1 ? kLast : 0) |
                                   (row_end && pwhole ? kWhole : 0));
    }
    if (fresh) {
      window();
      fresh = false;
    }
    do {
      if (ppg - bt_base >= 32) {
        bt_base += 32;
        window();
      }
      const unsigned long long src = __shfl_sync(0xffffffffu, bt_rows, ppg - bt_base) +
                                     static_cast<unsigned int>(poff * ROW);
      const int rows = min(p.bs - poff, todo);
      if (leader) {
        bulk_g2s(dst, reinterpret_cast<const void*>(src), rows * ROW, bar);
        bulk_g2s(dst + C::KV, reinterpret_cast<const void*>(src + v_less_k), rows * ROW, bar);
      }
      dst += rows * ROW;
      todo -= rows;
      poff += rows;
      if (poff == p.bs) {
        poff = 0;
        ++ppg;
      }
    } while (todo > 0);
    p_slot = p_slot + 1 == C::STAGES ? 0 : p_slot + 1;
    ++ahead;
    --left;
    pfirst = false;
    ++pst;
    if (!JOIN && row_end && left > 0) {
      pst = 0;
      if (++pkvh == p.hkv) {
        pkvh = 0;
        do ++pb; while (prefix[pb + 1] == prefix[pb]);  // left > 0: one with stages follows
        pnst = prefix[pb + 1] - prefix[pb];
      }
      open_row();
    }
    __syncwarp();
  };

  // ---------------------------------------------------------- consumer state
  // Fragments (lane = 4 g4 + t4): B of S^T: head g4, dims 32 w + 8 t4 + e; D of
  // S^T: tokens of rows g4 and g4 + 8, heads 2 t4 and 2 t4 + 1; D of O^T: of group
  // w columns 32 w + 4 g4 + {0, 2} (acc[w][0]) and {1, 3} (acc[w][1], times 16),
  // the same heads. Row r of a 16-token tile is token tau(r):
  //     tau(2 i) = 2 i, tau(2 i + 1) = (2 i + 4) % 8 + 8, tau(r + 8) = tau(r) + 1,
  // which makes the loads of 80-byte rows free of bank conflicts, K (8 lanes: two
  // rows 4 or 12 apart) as well as V (16 lanes: four even or four odd rows).
  uint32_t qf[NG][4];  // b0, b1 of the codes in bits 0-3, then of those in bits 4-7
  uint32_t qs[2];      // B of the lows' product: the groups' sums of q
  float f[2];          // scale * log2(e) over q's power of two, per head
  float m[2], l[2];    // running maximum; this lane's share of the sum, times 2^up
  int up = 14;         // P is held times 2^up
  float acc[NG][2][4], z[4];
  float* sc = nullptr;  // SCORED: the scores of the stage's first token
  const int tok_k = (g4 & 1) ? ((g4 + 3) & 7) + 8 : g4;  // tau(g4)
  const int tok_v = ((2 * t4 + 4) & 7) + 8;              // tau(2 t4 + 1)

  // The centring operand, by way of shared memory: an operand that the compiler knows to
  // be constant it writes out, four moves, before each of its products.
  uint32_t ca[4];
  load_words<4>(ca, smem + C::CENTRE_OFF);

  auto load_q = [&](int b, int kvh) {
    const bool real = g4 < p.group;
    const T* src = static_cast<const T*>(p.q) +
                   (static_cast<size_t>(b) * p.hq + kvh * p.group + g4) * D + 8 * t4;
    uint4 raw[NG];
#pragma unroll
    for (int w = 0; w < NG; ++w)
      raw[w] = real ? *reinterpret_cast<const uint4*>(src + 32 * w) : make_uint4(0u, 0u, 0u, 0u);
    float big = 0.f;
#pragma unroll
    for (int w = 0; w < NG; ++w)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        big = fmaxf(big, fabsf(to_f32(reinterpret_cast<const T*>(&raw[w])[e])));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    // k: big * 2^k in [2^7, 2^8); 0 for a zero or infinite q.
    const int e8 = (__float_as_int(big) >> 23) & 255;
    const int k = big == 0.f || e8 == 255 ? 0 : min(134 - e8, 126);
    const float up = pow2i(k);
    float sums[NG];
#pragma unroll
    for (int w = 0; w < NG; ++w) {
      float x[8];
      sums[w] = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = to_f32(reinterpret_cast<const T*>(&raw[w])[e]) * up;
        sums[w] += x[e];
      }
      qf[w][0] = pack_half2(x[0], x[4]);
      qf[w][1] = pack_half2(x[2], x[6]);
      qf[w][2] = pack_half2(x[1] * 0.0625f, x[5] * 0.0625f);
      qf[w][3] = pack_half2(x[3] * 0.0625f, x[7] * 0.0625f);
      sums[w] += __shfl_xor_sync(0xffffffffu, sums[w], 1);
      sums[w] += __shfl_xor_sync(0xffffffffu, sums[w], 2);
    }
    // The lows' product: its A has the lows of groups 0, 1 in every pair of k slots
    // below 8 and those of groups 2, 3 in every pair above; its B has the groups'
    // sums of q, rounded to fp16, in the first pair (lane t4 = 0), what that left over
    // in the second, and zeros in the others.
#pragma unroll
    for (int i = 0; i < NG / 2; ++i) {
      const float h0 = __half2float(__float2half_rn(sums[2 * i]));
      const float h1 = __half2float(__float2half_rn(sums[2 * i + 1]));
      qs[i] = t4 == 0   ? pack_half2(h0, h1)
              : t4 == 1 ? pack_half2(sums[2 * i] - h0, sums[2 * i + 1] - h1)
                        : 0u;
    }
    const float fh = p.scale_log2 * pow2i(-k);
    f[0] = __shfl_sync(0xffffffffu, fh, 8 * t4);
    f[1] = __shfl_sync(0xffffffffu, fh, 8 * t4 + 4);
  };

  auto consume = [&]() -> bool {
    const int4 md = meta[c_slot];
    const uint8_t* kst = ring + c_slot * C::STAGE;
    uint8_t* vst = ring + c_slot * C::STAGE + C::KV;
    const int nt = md.w & kTokens;
    if (md.w & kFirst) {
      load_q(md.x, md.y);
      up = 14;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
#pragma unroll
      for (int w = 0; w < NG; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[w][0][i] = acc[w][1][i] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] = 0.f;
    }
    if constexpr (SCORED)
      sc = p.scores + ((static_cast<size_t>(md.x) * p.hkv + md.y) * p.max_ctx + md.z) * p.gp;
    const bool ok = mbar_wait(full + c_slot, c_parity, abort_flag, p.status, kSiteKv4Wait,
                              p.timeout_ns);
    if (!__all_sync(0xffffffffu, ok)) return false;

    // The exponent of the largest scale of V in the stage, at least 1's. (A NaN scale is
    // passed over: its own columns are NaN whatever the others are multiplied by.)
    float less;  // what `up` goes down by, negative
    {
      __half2 top = __half2half2(__ushort_as_half(0));
#pragma unroll
      for (int r0 = 0; r0 < kTok; r0 += 32) {
        if (r0 + lane < nt) {
          uint32_t par[NG / 2];
          load_words<NG / 2>(par, vst + (r0 + lane) * ROW + CODES);
#pragma unroll
          for (int w = 0; w < NG / 2; ++w) {
            const uint32_t size = par[w] & 0x7fff7fffu;
            top = __hmax2(top, *reinterpret_cast<const __half2*>(&size));
          }
        }
      }
      const uint32_t bits = *reinterpret_cast<const uint32_t*>(&top);
      const uint32_t big = __reduce_max_sync(0xffffffffu, max(bits & 0xffffu, bits >> 16));
      const int now = min(up, 14 - (max(static_cast<int>(big >> 10), 15) - 15));
      less = static_cast<float>(now - up);
      up = now;
    }

    // Scores of the stage's tokens: s[i][0..1] token 16 i + tok_k, s[i][2..3] the
    // token after it.
    float s[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const uint8_t* ra = kst + (16 * i + tok_k) * ROW;
      const uint8_t* rb = ra + ROW;
      uint32_t xa[NG], xb[NG];
      load_words<NG>(xa, ra + 4 * NG * t4);
      load_words<NG>(xb, rb + 4 * NG * t4);
      uint32_t sa[NG], sb[NG];  // scales, then lows
      load_words<NG>(sa, ra + CODES);
      load_words<NG>(sb, rb + CODES);
      float lows[4];
      if constexpr (NG == 4)
        mma_k16_new(lows, sa[2], sb[2], sa[3], sb[3], qs[0], qs[1]);
      else
        mma_k8_new(lows, sa[1], sb[1], qs[0]);
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NG; ++w) {
        float d[4];
        const uint32_t ya = xa[w] >> 8, yb = xb[w] >> 8;
        mma_k16_new(d, xa[w] & 0x000F000Fu, xb[w] & 0x000F000Fu, ya & 0x000F000Fu, yb & 0x000F000Fu,
                qf[w][0], qf[w][1]);
        mma_k16(d, xa[w] & 0x00F000F0u, xb[w] & 0x00F000F0u, ya & 0x00F000F0u, yb & 0x00F000F0u,
                qf[w][2], qf[w][3]);
        const __half2 pa = *reinterpret_cast<const __half2*>(&sa[w / 2]);
        const __half2 pb = *reinterpret_cast<const __half2*>(&sb[w / 2]);
        const float fa = w % 2 == 0 ? __low2float(pa) : __high2float(pa);
        const float fb = w % 2 == 0 ? __low2float(pb) : __high2float(pb);
        sum[0] = fmaf(fa, d[0], sum[0]);
        sum[1] = fmaf(fa, d[1], sum[1]);
        sum[2] = fmaf(fb, d[2], sum[2]);
        sum[3] = fmaf(fb, d[3], sum[3]);
      }
      const uint64_t f2 = f2_pack(f[0], f[1]), up = f2_pack(0x1p24f, 0x1p24f);
#pragma unroll
      for (int c = 0; c < 4; c += 2)
        f2_unpack(f2_mul(f2_fma(f2_pack(sum[c], sum[c + 1]), up, f2_pack(lows[c], lows[c + 1])), f2),
                  s[i][c], s[i][c + 1]);
    }
    if (nt < kTok) {
      // Past the last token: no score; the ring's old bytes there must not reach
      // the products as a NaN scale or low either.
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (16 * i + tok_k + (c >> 1) >= nt) s[i][c] = -INFINITY;
      for (int r = nt + lane; r < kTok; r += 32) {
        uint32_t* par = reinterpret_cast<uint32_t*>(vst + r * ROW + CODES);
#pragma unroll
        for (int w = 0; w < NG; ++w) par[w] = 0u;
      }
      __syncwarp();
    }
    if constexpr (SCORED) {
      if (2 * t4 < p.gp) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int tok = 16 * i + tok_k + h;
            if (tok < nt) {
              if (p.gp == 1)
                sc[tok] = s[i][2 * h];
              else
                *reinterpret_cast<float2*>(sc + tok * p.gp + 2 * t4) =
                    make_float2(s[i][2 * h], s[i][2 * h + 1]);
            }
          }
      }
    }
    // Online softmax: per head the maximum over the 8 lanes of its scores.
    float alpha[2], shift[2];  // shift: up - m
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float mx = fmaxf(s[0][h], s[0][h + 2]);
#pragma unroll
      for (int i = 1; i < MT; ++i) mx = fmaxf(mx, fmaxf(s[i][h], s[i][h + 2]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
      mx = fmaxf(mx, m[h]);
      alpha[h] = fast_exp2(m[h] - mx + less);
      m[h] = mx;
      shift[h] = static_cast<float>(up) - mx;
    }
    // P^T as B fragments: tokens of rows 2 t4, 2 t4 + 1 (+ 8), head g4; and what rounding
    // it to fp16 left over.
    uint32_t pf[MT][2], pl[MT][2];
    uint64_t add = f2_pack(0.f, 0.f);
    const uint64_t sh = f2_pack(shift[0], shift[1]);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float e0, e1;
        f2_unpack(f2_add(f2_pack(s[i][2 * c], s[i][2 * c + 1]), sh), e0, e1);
        e0 = fast_exp2(e0);
        e1 = fast_exp2(e1);
        add = f2_add(add, f2_pack(e0, e1));
        const uint32_t hi = pack_half2(e0, e1);
        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        float r0, r1;
        f2_unpack(f2_fma(f2_pack(back.x, back.y), f2_pack(-1.f, -1.f), f2_pack(e0, e1)), r0, r1);
        pf[i][c] = transpose8(hi);
        pl[i][c] = transpose8(pack_half2(r0, r1));
      }
    }
    float add0, add1;
    f2_unpack(add, add0, add1);
    l[0] = fmaf(l[0], alpha[0], add0);
    l[1] = fmaf(l[1], alpha[1], add1);
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
      for (int w = 0; w < NG; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[w][0][i] *= alpha[i & 1];
          acc[w][1][i] *= alpha[i & 1];
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] *= alpha[i & 1];
    }
    // O^T += V^T P^T. centre: - c P scale of the stage, the same in every column.
    float centre[NG][4];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const uint8_t* ra = vst + (16 * i + 2 * t4) * ROW;  // rows 2 t4 and (below, + ROW) 2 t4 + 8
      const uint8_t* rb = vst + (16 * i + tok_v) * ROW;   // rows 2 t4 + 1 and 2 t4 + 9
      uint32_t va[NG / 2], vb[NG / 2], vc[NG / 2], vd[NG / 2];
      load_words<NG / 2>(va, ra + 2 * NG * g4);
      load_words<NG / 2>(vb, rb + 2 * NG * g4);
      load_words<NG / 2>(vc, ra + ROW + 2 * NG * g4);
      load_words<NG / 2>(vd, rb + ROW + 2 * NG * g4);
      uint32_t sa[NG], sb[NG], sc2[NG], sd[NG];  // scales, then lows
      load_words<NG>(sa, ra + CODES);
      load_words<NG>(sb, rb + CODES);
      load_words<NG>(sc2, ra + ROW + CODES);
      load_words<NG>(sd, rb + ROW + CODES);
      // P . (low + c scale): row g4 has the middles of group g4 % 2, row g4 + 8 those
      // of group 2 + g4 % 2.
      const uint32_t pick = (g4 & 1) ? 0x7632u : 0x5410u;
      constexpr int L = NG / 2;
      uint32_t ma[2], mb[2], mc[2], md2[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int k = j * (L - 1);
        ma[j] = hfma2(sa[k], kEight, sa[L + k]);
        mb[j] = hfma2(sb[k], kSeven, sb[L + k]);
        mc[j] = hfma2(sc2[k], kEight, sc2[L + k]);
        md2[j] = hfma2(sd[k], kSeven, sd[L + k]);
      }
      const uint32_t z0 = __byte_perm(ma[0], mb[0], pick), z1 = __byte_perm(ma[1], mb[1], pick);
      const uint32_t z2 = __byte_perm(mc[0], md2[0], pick), z3 = __byte_perm(mc[1], md2[1], pick);
      mma_k16(z, z0, z1, z2, z3, pf[i][0], pf[i][1]);
      mma_k16(z, z0, z1, z2, z3, pl[i][0], pl[i][1]);
#pragma unroll
      for (int w = 0; w < NG; ++w) {
        const uint32_t half = w % 2 == 0 ? 0x5410u : 0x7632u;
        const uint32_t s0 = __byte_perm(sa[w / 2], sb[w / 2], half);
        const uint32_t s1 = __byte_perm(sc2[w / 2], sd[w / 2], half);
        const uint32_t b0 = hfma2(pf[i][0], s0, hmul2(pl[i][0], s0));
        const uint32_t b1 = hfma2(pf[i][1], s1, hmul2(pl[i][1], s1));
        const uint32_t x = __byte_perm(va[w / 2], vb[w / 2], half);
        const uint32_t y = __byte_perm(vc[w / 2], vd[w / 2], half);
        const uint32_t x8 = x >> 8, y8 = y >> 8;
        if (i == 0)
          mma_k16_new(centre[w], ca[0], ca[1], ca[2], ca[3], b0, b1);
        else
          mma_k16(centre[w], ca[0], ca[1], ca[2], ca[3], b0, b1);
        mma_k16(acc[w][0], x & 0x000F000Fu, x8 & 0x000F000Fu, y & 0x000F000Fu, y8 & 0x000F000Fu,
                b0, b1);
        mma_k16(acc[w][1], x & 0x00F000F0u, x8 & 0x00F000F0u, y & 0x00F000F0u, y8 & 0x00F000F0u,
                b0, b1);
      }
    }
#pragma unroll
    for (int w = 0; w < NG; ++w) {
      const uint64_t c2 = f2_pack(centre[w][0], centre[w][1]), up = f2_pack(16.f, 16.f);
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        f2_unpack(f2_add(f2_pack(acc[w][0][i], acc[w][0][i + 1]), c2), acc[w][0][i],
                  acc[w][0][i + 1]);
        f2_unpack(f2_fma(c2, up, f2_pack(acc[w][1][i], acc[w][1][i + 1])), acc[w][1][i],
                  acc[w][1][i + 1]);
      }
    }
    if (md.w & kLast) {
      const int pair = md.x * p.hkv + md.y;
      const size_t slot0 = (static_cast<size_t>(worker) + pair) * p.group;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], o);
        const float inv = 1.f / l[h];
        const int head = 2 * t4 + h;
        const size_t row = static_cast<size_t>(pair) * p.group + head, pr = slot0 + head;
#pragma unroll
        for (int w = 0; w < NG; ++w) {
          const float low = __shfl_sync(0xffffffffu, z[h + 2 * (w / 2)], 4 * (w % 2) + t4);
          float o[4];
          o[0] = fmaf(acc[w][0][h], 0x1p24f, low) * inv;
          o[1] = fmaf(acc[w][1][h], 0x1p20f, low) * inv;
          o[2] = fmaf(acc[w][0][h + 2], 0x1p24f, low) * inv;
          o[3] = fmaf(acc[w][1][h + 2], 0x1p20f, low) * inv;
          const int col = 32 * w + 4 * g4;
          if constexpr (JOIN) {
            // The ring holds no copy any more: this was the warp's last stage.
            *reinterpret_cast<float4*>(ring + (head * D + col) * 4) =
                make_float4(o[0], o[1], o[2], o[3]);
          } else if (head < p.group) {
            if (md.w & kWhole)
              *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + row * D + col) =
                  make_uint2(pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3]));
            else
              *reinterpret_cast<float4*>(p.o_part + pr * D + col) =
                  make_float4(o[0], o[1], o[2], o[3]);
          }
        }
        // A part whose scores are all NaN has no maximum, yet is not an empty one.
        const float mh = l[h] != l[h] ? fmaxf(m[h], 0.f) : m[h];
        if constexpr (JOIN) {
          if (g4 == 0)
            *reinterpret_cast<float2*>(ring + C::ML_OFF + head * 8) = make_float2(mh, pow2i(-up) * l[h]);
        } else if (head < p.group && g4 == 0 && (SCORED || !(md.w & kWhole))) {
          p.m_part[pr] = mh;
          p.l_part[pr] = pow2i(-up) * l[h];
        }
      }
    }
    __syncwarp();
    --ahead;
    if (++c_slot == C::STAGES) {
      c_slot = 0;
      c_parity ^= 1u;
    }
    return true;
  };

  for (int i = 0; i < C::STAGES; ++i) produce();
  while (ahead > 0) {
    if (!consume()) break;
    // The slot just read is refilled by the async proxy.
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    produce();
  }
  // Never exit with a copy in flight (only reached with copies pending after a timeout).
  for (; ahead > 0; --ahead) {
    mbar_wait(full + c_slot, c_parity, nullptr, p.status, kSiteKv4Drain, p.timeout_ns);
    if (++c_slot == C::STAGES) {
      c_slot = 0;
      c_parity ^= 1u;
    }
  }
  if constexpr (JOIN) {
    // o = sum_w l_w 2^(m_w - M) o_w / L, L = sum_w l_w 2^(m_w - M), M the largest m_w;
    // the first runs.workers warps have parts. An empty sequence has none: zeros.
    float2* total = reinterpret_cast<float2*>(smem + C::PREFIX_OFF);  // M and 1 / L per head
    const int kvh = static_cast<int>(blockIdx.x) - my_b * p.hkv;
    const int parts = static_cast<int>(runs.workers);
    __syncthreads();
    for (int x = threadIdx.x; x < p.group * (D / 2); x += C::THREADS) {
      const int head = x / (D / 2), col = 2 * (x % (D / 2));
      const uint8_t* ml = smem + C::ML_OFF + head * 8;
      float big = -INFINITY;
      for (int w = 0; w < parts; ++w)
        big = fmaxf(big, *reinterpret_cast<const float*>(ml + w * C::RING));
      float den = 0.f, n0 = 0.f, n1 = 0.f;
      for (int w = 0; w < parts; ++w) {
        const float2 mw = *reinterpret_cast<const float2*>(ml + w * C::RING);
        const float2 o = *reinterpret_cast<const float2*>(smem + w * C::RING + (head * D + col) * 4);
        const float e = mw.y * fast_exp2(mw.x - big);
        den += e;
        n0 = fmaf(e, o.x, n0);
        n1 = fmaf(e, o.y, n1);
      }
      const float inv = parts == 0 ? 0.f : 1.f / den;
      if (SCORED && col == 0) total[head] = make_float2(big, inv);
      *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) +
                                   (static_cast<size_t>(my_b) * p.hq + kvh * p.group + head) * D +
                                   col) = pack2<T>(n0 * inv, n1 * inv);
    }
    if constexpr (SCORED) {
      // Each token's weight, summed over the heads, to its slot's total.
      __syncthreads();
      const float* row = p.scores + static_cast<size_t>(blockIdx.x) * p.max_ctx * p.gp;
      for (int t = threadIdx.x; t < my_len; t += C::THREADS) {
        float w = 0.f;
        for (int g = 0; g < p.group; ++g)
          w = fmaf(fast_exp2(row[t * p.gp + g] - total[g].x), total[g].y, w);
        const int in = p.by_bs.quotient(t);
        const int page = p.bt[static_cast<size_t>(my_b) * p.max_blocks + in];
        // A page outside the cache was reported where its rows were to be read.
        if (static_cast<unsigned>(page) < static_cast<unsigned>(p.num_blocks))
          atomicAdd(p.weights + (static_cast<size_t>(page) * p.hkv + kvh) * p.bs + (t - in * p.bs),
                    w);
      }
    }
  }
}

size_t align256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

// Workspace of one launch (launches of one call follow each other in the stream
// and use the same): parts of every resident warp and every (sequence, kv head).
struct Workspace {
  int* first;
  float *o, *m, *l, *scores;
  size_t bytes;
};

// Resident warps the workspace has room for: of 160 SMs, more than a B200 has, so
// that its size goes by the call's sizes alone.
constexpr int64_t kMaxWorkers = 160 * std::max(Kv4Cfg<64>::W, Kv4Cfg<128>::W);

Workspace carve(void* base, int64_t batch, int64_t hq, int64_t hkv, int64_t d, size_t score_bytes) {
  uint8_t* b = static_cast<uint8_t*>(base);
  const int64_t nb = std::min<int64_t>(batch, kLaunchBatch);
  const size_t rows = static_cast<size_t>(kMaxWorkers + nb * hkv) * (hq / hkv);
  const size_t fb = align256(static_cast<size_t>(nb + 1) * 4);
  const size_t ob = align256(rows * d * 4);
  const size_t ml = align256(rows * 4);
  Workspace w;
  w.first = reinterpret_cast<int*>(b);
  w.o = reinterpret_cast<float*>(b + fb);
  w.m = reinterpret_cast<float*>(b + fb + ob);
  w.l = reinterpret_cast<float*>(b + fb + ob + ml);
  w.scores = reinterpret_cast<float*>(b + fb + ob + 2 * ml);
  w.bytes = fb + ob + 2 * ml + align256(score_bytes);
  return w;
}

template <int D, typename T, bool SCORED, bool JOIN>
cudaError_t launch_kernel(const Kv4DecParams& p, int grid, const LaunchCtx& ctx) {
  using C = Kv4Cfg<D>;
  auto kern = kv4_decode_kernel<D, T, SCORED, JOIN>;
  static SmemLimit limit;
  cudaError_t e = allow_smem(kern, C::SMEM, limit);
  if (e != cudaSuccess) return e;
  kern<<<grid, C::THREADS, C::SMEM, ctx.stream>>>(p);
  return cudaGetLastError();
}

template <int D, typename T>
cudaError_t dispatch(const Kv4DecParams& p, int grid, bool join, const LaunchCtx& ctx) {
  if (join)
    return p.scores != nullptr ? launch_kernel<D, T, true, true>(p, grid, ctx)
                               : launch_kernel<D, T, false, true>(p, grid, ctx);
  return p.scores != nullptr ? launch_kernel<D, T, true, false>(p, grid, ctx)
                             : launch_kernel<D, T, false, false>(p, grid, ctx);
}

}  // namespace

size_t kv4_decode_workspace_bytes(int64_t batch, int64_t hq, int64_t hkv, int64_t d, int64_t max_ctx,
                                  bool weights) {
  const int64_t nb = std::min<int64_t>(batch, kLaunchBatch);
  return carve(nullptr, batch, hq, hkv, d,
               weights ? score_bytes(nb, hkv, hq / hkv, max_ctx) : 0).bytes;
}

cudaError_t launch_kv4_decode(const Kv4DecodeArgs& a, const LaunchCtx& ctx) {
  const int64_t group = a.hq / a.hkv;
  const bool scored = a.weights != nullptr;
  if (a.max_ctx == 0)
    return cudaMemsetAsync(a.out, 0, static_cast<size_t>(a.batch) * a.hq * a.d * 2, ctx.stream);
  Workspace w = carve(a.workspace, a.batch, a.hq, a.hkv, a.d, 0);
  const int64_t warps = a.d == 64 ? Kv4Cfg<64>::W : Kv4Cfg<128>::W;
  const int64_t tok = a.d == 64 ? Kv4Cfg<64>::TOK : Kv4Cfg<128>::TOK;
  for (int64_t b0 = 0; b0 < a.batch; b0 += kLaunchBatch) {
    const int64_t nb = std::min<int64_t>(kLaunchBatch, a.batch - b0);
    const int64_t row_bytes = a.d / 2 + a.d / 8, row0 = b0 * a.hq;
    Kv4DecParams p;
    p.q = static_cast<const uint8_t*>(a.q) + row0 * a.d * 2;
    p.kc = static_cast<const uint8_t*>(a.k_cache);
    p.vc = static_cast<const uint8_t*>(a.v_cache);
    p.bt = a.block_tables + b0 * a.max_blocks;
    p.ctx = a.context_lens + b0;
    p.out = static_cast<uint8_t*>(a.out) + row0 * a.d * 2;
    p.o_part = w.o;
    p.m_part = w.m;
    p.l_part = w.l;
    p.first = w.first;
    p.gp = static_cast<int>(score_heads(group));
    p.scores = scored ? w.scores : nullptr;
    p.weights = a.weights;
    p.by_bs = FastDiv(a.bs);
    p.status = ctx.status;
    p.timeout_ns = ctx.timeout_ns;
    p.block_stride = static_cast<unsigned int>(a.hkv * a.bs * row_bytes);
    p.batch = static_cast<int>(nb);
    p.hq = static_cast<int>(a.hq);
    p.hkv = static_cast<int>(a.hkv);
    p.group = static_cast<int>(group);
    p.bs = static_cast<int>(a.bs);
    p.max_blocks = static_cast<int>(a.max_blocks);
    p.num_blocks = static_cast<int>(a.num_blocks);
    p.max_ctx = static_cast<int>(a.max_ctx);
    p.scale_log2 = a.scale * kLog2e;
    // One CTA per SM, or one per stage when there cannot be that many; or one per row
    // (JOIN), in one launch, where that makes no warp's chain of stages longer: no more
    // rows than SMs, at most two stages a warp and no more than equal runs over all
    // resident warps would give. (Equal runs and finish / JOIN, us, 8 kv heads of 4 query
    // heads, head_dim 128: 1 x 64 tokens 7.4 / 4.6, 8 x 200 9.0 / 5.6, 18 x 576
    // 11.3 / 7.7, 18 x 1152 14.7 / 10.8, with weights 16.5 / 13.1; outside the rule
    // 1 x 1152 8.8 / 9.6, 8 x 2304 14.1 / 15.3, 24 x 576 12.8 / 13.8.)
    const int64_t row_stages = (a.max_ctx + tok - 1) / tok, stages = nb * a.hkv * row_stages;
    const int64_t chain = (row_stages + warps - 1) / warps, resident = ctx.sm_count * warps;
    const bool join = nb * a.hkv <= ctx.sm_count && chain <= 2 &&
                      chain <= std::max<int64_t>(1, (stages + resident - 1) / resident);
    const int grid = static_cast<int>(
        join ? nb * a.hkv
             : std::min<int64_t>(std::min<int64_t>(ctx.sm_count, kMaxWorkers / warps), stages));
    cudaError_t e;
    if (a.d == 64)
      e = a.bf16 ? dispatch<64, __nv_bfloat16>(p, grid, join, ctx) : dispatch<64, __half>(p, grid, join, ctx);
    else
      e = a.bf16 ? dispatch<128, __nv_bfloat16>(p, grid, join, ctx) : dispatch<128, __half>(p, grid, join, ctx);
    if (e != cudaSuccess) return e;
    if (join) continue;
    FinishArgs f;
    f.o = w.o;
    f.m = w.m;
    f.l = w.l;
    f.context_lens = p.ctx;
    f.first = w.first;
    f.workers = static_cast<int64_t>(grid) * warps;
    f.partition = tok;
    f.parts = 0;
    f.scores = p.scores;
    f.weights = a.weights;
    f.block_tables = p.bt;
    f.out = p.out;
    f.bf16 = a.bf16;
    f.batch = nb;
    f.hq = a.hq;
    f.hkv = a.hkv;
    f.d = a.d;
    f.bs = a.bs;
    f.num_blocks = a.num_blocks;
    f.max_blocks = a.max_blocks;
    f.max_ctx = a.max_ctx;
    e = launch_finish(f, ctx);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace fab
