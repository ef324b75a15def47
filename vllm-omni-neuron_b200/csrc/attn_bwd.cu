// Attention's backward pass for sm_100a, which recomputes the probabilities from the forward's log-sum-exp:
//     P = exp(scale Q K^T - lse)            dV = P^T dO
//     dS = P (dO V^T - delta)               delta = rowsum(dO O) - dlse, as the derivative of lse is P
//     dQ = scale dS K                       dK = scale dS^T Q
// The forward's lse is the one of ring_attention_const_max_fwd(training=True)
// (vllm_omni_neuron/kernels/nkilib/experimental/attention/ring_attention_const_max_fwd.py:1062-1065), so the gradients
// of a part of the keys are those of that part of the whole softmax, and parts add up.
//
// Two kinds of CTA pairs, one per side of the score matrix, so that every gradient is summed in one CTA pair's TMEM
// in a fixed order and written once: no atomics, no fp32 gradient in HBM, the same bits every time. The price is
// that S and dP are formed twice: 7 matrix products instead of the 5 of one pass that adds dQ with atomics.
//   dkdv: a pair of CTAs holds 256 keys of one key head (128 rows of TMEM in each) and walks the query tiles of every
//         query head that shares it: S^T = K Q^T, dP^T = V dO^T, then dV += P^T dO and dK += dS^T Q with P^T, dS^T
//         read straight from TMEM.
//   dq:   a pair holds 256 queries of one head and walks the key tiles: S = Q K^T, dP = dO V^T, dQ += dS K.
// Both use tcgen05 cta_group::2 (M = 256, N = 128): each CTA stages half of every streamed operand, split by rows for
// the S and dP products and by head dimension for the others, as a one-CTA M = 128 product would need 128 B of
// shared-memory operands a clock and leave no room for the loads.
// Warps: 0 TMA producer, 1 and 2 MMA issuers (the even CTA's), 4..19 exponentials and gradients of the scores: a thread
// owns one TMEM lane (a key in dkdv, a query in dq), warpgroup wg the columns [32 wg, 32 wg + 32).
// A wait costs an issuer some 170 to 300 clocks after its last MMA, and the tensor pipe queues about one, so each issuer
// waits once a step: on one barrier that counts the score warps' arrivals and the bytes of every operand of that step.
// The products that depend on different events are issued by different warps, so that one's wait is filled with the
// other's products: issuer X the gradients and the scores that follow them in the same TMEM columns, issuer Y dP. The pipe takes
// two issuers' products in turn, so X lets Y's batch go ahead where the score warps need it first.
// Matrix products per 128 x 128 scores of a CTA: 512 clocks each; exponentials: 1024 clocks of the MUFU unit.
// Measured, clocks a step of a pair at 32760 tokens: dkdv 2450 (its products alone 2180), dq 2250 (1540), at which the GPU is at
// its power cap (1.59 to 1.75 GHz). Over several GPUs, among other passes and alone: 4096 tokens x 40 heads 0.94 to 1.09 ms (788 to 914
// TFLOP/s of the 5 products, 1.1 to 1.3 PFLOP/s of the 7), 32760 x 8 heads 11.3 to 11.9 ms (924 to 972), 8190 x 512 x 40 heads 0.36 to
// 0.39 ms, 0.41 to 0.46 with a cold L2.
//
// Rounding: P and dS are rounded to bf16 as tensor-core operands (2^-8 relative each, at most); everything else is fp32 until the
// gradients are rounded once.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "host_util.h"

namespace vomni {
namespace abwd {

constexpr int kD = 128;
constexpr int kTile = 128;              // columns of a step (queries in dkdv, keys in dq); rows of a CTA
constexpr int kGroups = 4;              // score warpgroups: each owns kCols columns of a step's scores
constexpr int kCols = kTile / kGroups;  // 32: one TMEM load
constexpr int kControl = 4;             // warps ahead of them: TMA producer, two MMA issuers, one idle
constexpr int kThreads = 32 * kControl + 128 * kGroups;
// Batch elements of a launch with lengths of their own: more run as launches one after another, each with its own tail (the split rule
// looks at the batch as one launch).
constexpr int kMaxSeqs = 16;
constexpr uint32_t kBox = 64 * 64 * 2;  // 8 KB: one TMA box, 64 rows x 64 dims, 128-byte swizzled
constexpr uint32_t kTileBytes = 4 * kBox;  // resident operand: [2 dim halves][2 row halves] boxes
constexpr uint32_t kHalfTile = 2 * kBox;   // a CTA's half of a streamed operand
constexpr float kNoKeys = 1e30f;        // -lse / scale of a row without keys (its sign that of -scale): no probabilities
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kScoreWarps = 8 * kGroups;  // score warps of both CTAs: arrivals per READY phase

// One set of maps for a batch of equal lengths (the batch element is a coordinate), or one per batch element
// whose extents end at its lengths: rows behind them read as zero, whatever they hold.
template <int N>
struct Maps {
  CUtensorMap q[N], k[N], v[N], d_o[N];
  CUtensorMap stats;  // Params::stats as [b * hq * rows][8]
};

struct Params {
  int b0;                     // first batch element of this launch
  int s_q, s_kv, hq, hkv, group;
  int q_len[kMaxSeqs], kv_len[kMaxSeqs];  // of each batch element (of the launch); [0] for all in a uniform one
  int rows;                   // row pitch of stats: s_q rounded up to whole tiles
  const uint4* stats;         // [b * hq, rows]: -lse / scale and -delta, three bf16 pieces each (stats_of)
  float scale, scale_log2;
  // The launch's CTA pairs: the dK/dV ones first (they walk longer), then the dQ ones. A walk's tiles are dealt to
  // splits of `per` tiles.
  int k_pairs;                // pairs of 256 keys, over all key heads, batch elements and splits
  int k_tiles2, q_tiles2;     // 256-row tiles of a head's keys / queries
  int k_splits, k_per, q_splits, q_per;
  void *dq, *dk, *dv;         // bf16 [b, s, heads, 128], or, where split, fp32 parts [split][b, s, heads, 128]
  long long q_part, k_part;   // elements of one part
  int* status;
};

// Device status sites (VOMNI_DEV_TIMEOUT_BASE + site).
enum Site : int { kSiteProducer = 0x10, kSiteMma = 0x11, kSiteScores = 0x12, kSiteOut = 0x13, kSiteDrain = 0x14, kSiteRows = 0x15 };

// mbar_wait whose thread is suspended for 40 ns at a time at most (without the hint it wakes some hundred clocks late), and
// looks at the abort flag and the clock once in 64 polls.
VOMNI_DEV bool mbar_poll(uint64_t* bar, uint32_t parity, volatile int* abort, int* status, int code) {
  const uint32_t addr = smem_u32(bar);
  uint64_t t0 = 0;
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i) {
      uint32_t ok;
      asm volatile(
          "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 40;\n\tselp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(ok)
          : "r"(addr), "r"(parity)
          : "memory");
      if (ok) return true;
    }
    if (*abort) return false;
    const uint64_t t = globaltimer();
    if (t0 == 0) t0 = t;
    if (t - t0 > kWaitBudgetNs) {
      *abort = 1;
      if (status) atomicCAS(status, 0, code);
      return false;
    }
  }
}

// The issuers poll; the others may be suspended for longer, which leaves them the issue slots. (32760 tokens, clocks a step:
// dkdv 2590 with polling score warps, 2460 with suspended ones; dq 2320 and 2790, so its score warps poll. Polling with
// test_wait, which never suspends: 2500 and 2380.)
VOMNI_DEV bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort, int* status, int site) {
  const int code = VOMNI_DEV_TIMEOUT_BASE + site;
  return site == kSiteMma ? mbar_poll(bar, parity, abort, status, code) : mbar_wait_spin(bar, parity, abort, status, code);
}

// P / dS in TMEM: the bf16 values of columns [16 kk, 16 kk + 16) sit in the 8 TMEM columns from pcol(kk). Each
// warpgroup writes over score columns that it has read itself.
__host__ __device__ constexpr uint32_t pcol(int kk) { return (kk >> 1) * kCols + (kk & 1) * 8; }

constexpr uint32_t kIdescScores = idesc_bf16(256, 128, false);
constexpr uint32_t kIdescGrad = idesc_bf16(256, 128, true);

// scores[256 x 128] = A (resident, 128 rows in each CTA) B^T (streamed, 64 rows in each CTA), both K-major over d; added to
// what the columns hold where `add`.
VOMNI_DEV void issue_scores(uint32_t d, uint64_t a, uint64_t b, bool add = false) {
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
    mma_f16_ss_pair(d, a + (((kk >> 2) * 2 * kBox + (kk & 3) * 32) >> 4), b + (((kk >> 2) * kBox + (kk & 3) * 32) >> 4),
                    kIdescScores, (kk > 0 || add) ? 1u : 0u);
}
// grad[256 x 128] += W (TMEM, 128 columns) B (streamed: 128 rows, 64 dims in each CTA, MN-major).
VOMNI_DEV void issue_grad(uint32_t d, uint32_t w, uint64_t b, bool accumulate) {
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
    mma_f16_ts_pair(d, w + pcol(kk), b + ((kk * 2048) >> 4), kIdescGrad, (kk > 0 || accumulate) ? 1u : 0u);
}
VOMNI_DEV uint64_t desc_k(const void* p) { return make_sdesc(smem_u32(p), 16, 1024, kLayoutSW128); }
VOMNI_DEV uint64_t desc_mn(const void* p) { return make_sdesc(smem_u32(p), kHalfTile, 1024, kLayoutSW128); }

// Loads of this CTA's rows of a resident operand (128 rows x 128 dims) and of its halves of a streamed one.
VOMNI_DEV void load_resident(const CUtensorMap* m, uint32_t bar, uint8_t* dst, int row, int h, int b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) tma_load_4d_pair(m, bar, dst + i * kBox, (i >> 1) * 64, row + (i & 1) * 64, h, b);
}
VOMNI_DEV void load_rows(const CUtensorMap* m, uint32_t bar, uint8_t* dst, int row, int h, int b, int rank) {
  tma_load_4d_pair(m, bar, dst, 0, row + rank * 64, h, b);
  tma_load_4d_pair(m, bar, dst + kBox, 64, row + rank * 64, h, b);
}
VOMNI_DEV void load_dims(const CUtensorMap* m, uint32_t bar, uint8_t* dst, int row, int h, int b, int rank) {
  tma_load_4d_pair(m, bar, dst, rank * 64, row, h, b);
  tma_load_4d_pair(m, bar, dst + kBox, rank * 64, row + 64, h, b);
}

// One arrival of this warp on the leader's barrier: its loads from TMEM have completed (signal), or its stores too (publish).
VOMNI_DEV void signal(uint32_t bar_cluster) {
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive_cluster(bar_cluster);
}
VOMNI_DEV void publish(uint32_t bar_cluster) {
  tmem_st_wait();
  signal(bar_cluster);
}

// kCols columns of one row of a gradient (its fp32 sums, raw), times `scale`, to the output row (bf16, or fp32 parts).
VOMNI_DEV void store_share(const uint32_t (&o)[kCols], float scale, bool parts, void* out, long long at) {
  float v[kCols];
#pragma unroll
  for (int i = 0; i < kCols; ++i) v[i] = __uint_as_float(o[i]) * scale;
  if (parts) {
    float4* dst = reinterpret_cast<float4*>(static_cast<float*>(out) + at);
#pragma unroll
    for (int i = 0; i < kCols / 4; ++i) dst[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else {
    uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + at);
#pragma unroll
    for (int i = 0; i < kCols / 8; ++i)
      dst[i] = make_uint4(pack_bf16x2(v[8 * i], v[8 * i + 1]), pack_bf16x2(v[8 * i + 2], v[8 * i + 3]),
                          pack_bf16x2(v[8 * i + 4], v[8 * i + 5]), pack_bf16x2(v[8 * i + 6], v[8 * i + 7]));
  }
}
VOMNI_DEV void clear(uint32_t (&o)[kCols]) {
#pragma unroll
  for (int i = 0; i < kCols; ++i) o[i] = 0u;
}

// A CTA that gave up waits (bounded) for the copies it may still have in flight: barrier `bar` has had `uses` loads.
VOMNI_DEV void drain(uint64_t* bar, int uses, int* status, int code) {
  if (uses <= 0) return;
  int ignored = 0;
  mbar_wait(bar, (uses - 1) & 1, &ignored, status, code);
}

// A float as the sum of three bf16, exactly: each takes the 8 leading bits that are left, so that none is larger than the
// float and their sum, in any order, needs no more bits than it has. In the low halves of three words.
VOMNI_DEV void pieces_of(float v, uint32_t (&w)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const uint32_t h = __float_as_uint(v) & 0xffff0000u;
    w[i] = h >> 16;
    v -= __uint_as_float(h);
  }
}
VOMNI_DEV uint4 stats_of(float neg_lse_over_scale, float neg_delta) {
  uint32_t l[3], d[3];
  pieces_of(neg_lse_over_scale, l);
  pieces_of(neg_delta, d);
  return make_uint4(l[0] | l[1] << 16, l[2] | d[0] << 16, d[1] | d[2] << 16, 0);
}
// Back to -log2(e) lse and -delta.
VOMNI_DEV void sum_stats(const uint4& w, float scale_log2, float& nlse2, float& neg_delta) {
  auto lo = [](uint32_t u) { return __uint_as_float(u << 16); };
  auto hi = [](uint32_t u) { return __uint_as_float(u & 0xffff0000u); };
  nlse2 = (lo(w.x) + hi(w.x) + lo(w.y)) * scale_log2;
  neg_delta = hi(w.y) + lo(w.z) + hi(w.z);
}

// The shared prologue and epilogue of both kernels: barriers, TMEM, and their release.
VOMNI_DEV uint32_t open_cta(uint64_t* bars, int n, int counted0, int counted1, uint32_t* tmem_slot, volatile int* abort_flag) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < n; ++i) mbar_init(&bars[i], i >= counted0 && i < counted1 ? kScoreWarps + 1 : 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (threadIdx.x >> 5 == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  return *tmem_slot;
}
VOMNI_DEV void close_cta(uint32_t tbase) {
  tc_fence_before();
  cluster_sync();  // no CTA leaves while its pair may still touch its barriers or TMEM
  if (threadIdx.x >> 5 == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tbase, 512);
  }
}

// ================================================================ dK, dV
namespace dkdv {
// Streamed operands of a query tile, two slots each: Q and dO by rows (for S^T, dP^T), dO and Q by dims (for dV, dK).
constexpr uint32_t kSmemK = 0, kSmemV = kTileBytes, kSmemStream = 2 * kTileBytes;
constexpr int kSlots = 2, kLSlots = 4;
constexpr uint32_t smem_of(int kind, int step) { return kSmemStream + (kind * kSlots + (step & 1)) * kHalfTile; }
constexpr int kQr = 0, kOr = 1, kOd = 2, kQd = 3;
// A query's lse and delta belong to a column of the scores, so every thread would need them all: read from shared
// memory they took 1024 of the step's wavefronts, which the products' operands need (3650 clocks a step instead of 2670
// without them). They are added by the tensor cores instead, as one more step of 16 of each product: B holds the
// columns' pieces (stats, 16 bytes a query), A ones where the pieces are (columns 0-2 for S, 3-5 for dP) and zeros
// elsewhere. Unswizzled core matrices of 8 rows x 16 bytes; B's second half of the 16 is its first again, times zeros.
constexpr uint32_t kAuxBytes = 64 * 16, kOnesBytes = 128 * 32;
constexpr uint32_t kSmemAux = kSmemStream + 4 * kSlots * kHalfTile;  // [kLSlots] stats of this CTA's 64 queries of a step
constexpr uint32_t kSmemOnes = kSmemAux + kLSlots * kAuxBytes;       // A for S, A for dP
constexpr uint32_t kSmemBar = kSmemOnes + 2 * kOnesBytes;
constexpr uint32_t kSmemBytes = kSmemBar + 256 + 1024;
// TMEM columns: two score regions, dV, dK. Step j works in region j % 2, which holds S^T, then (once the score warps have
// read it) dP^T, then P^T and dS^T side by side, so that S^T of the next step is formed in the other one meanwhile.
constexpr uint32_t kColR = 0, kColDv = 256, kColDk = 384;
constexpr uint32_t kDs = kCols / 2;  // dS^T beside P^T: the second half of each warpgroup's columns

// Two barriers of a kind serve steps in turn; each is waited for before anything that its next phase depends on, so no
// wait can miss a phase. X issues dV(j), dK(j), S(j+2) in this order and MMAs of one thread complete in order, so S
// of step j complete frees the slots of dV(j-2) and dK(j-2) too.
enum Bar : int {
  START = 0,             // K and the first two tiles' Q rows and stats
  S_FULL = 1,            // + step % 2, as all below
  DP_FULL = S_FULL + 2,
  S_READ = DP_FULL + 2,  // Y's: the score warps hold S of step j; dO's rows of j (and V, for the first) are there
  PD_READY = S_READ + 2, // X's: P and dS of step j; dO's and Q's dims of j and Q's rows and stats of j + 2 are there
  OUT_FULL = PD_READY + 2,
  NBAR = OUT_FULL + 1
};
static_assert(NBAR * 8 + 8 <= 256, "barriers, TMEM slot and abort flag fit their area");

VOMNI_DEV uint64_t desc_aux(const void* p) { return make_sdesc(smem_u32(p), 0, 128, 0); }
VOMNI_DEV uint64_t desc_ones(const void* p) { return make_sdesc(smem_u32(p), 128, 256, 0); }

template <int N>
VOMNI_DEV void body(const Maps<N>& maps, const Params& p, uint8_t* smem, int pair) {
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kSmemBar);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kSmemBar + NBAR * 8 + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair_row = pair % p.k_tiles2 * 2 * kTile;
  const int row0 = pair_row + static_cast<int>(rank) * kTile;  // this CTA's first key
  const int hk = pair / p.k_tiles2 % p.hkv, z = pair / p.k_tiles2 / p.hkv;
  const int seq = z / p.k_splits, split = z % p.k_splits;
  const int mi = N == 1 ? 0 : seq, bz = N == 1 ? seq : 0, b = p.b0 + seq;
  const int q_len = p.q_len[mi], kv_len = p.kv_len[mi];
  const int q_tiles = (q_len + kTile - 1) / kTile;
  // this split's steps of the walk over (query head of the group, query tile)
  const int first = split * p.k_per;
  const int last = min(first + p.k_per, q_tiles * p.group);
  const int steps = pair_row < kv_len ? max(last - first, 0) : 0;

  if (steps > 0 && threadIdx.x < 256) {  // row threadIdx.x % 128 of one of the two A tiles of ones
    const int r = threadIdx.x & 127, which = threadIdx.x >> 7;
    uint4* row = reinterpret_cast<uint4*>(smem + kSmemOnes + which * kOnesBytes + (r >> 3) * 256 + (r & 7) * 16);
    constexpr uint32_t one = 0x3F80u;  // bf16 1
    row[0] = which ? make_uint4(0, one << 16, one | one << 16, 0) : make_uint4(one | one << 16, one, 0, 0);
    row[8] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  uint32_t tbase = 0;
  if (steps > 0)
    tbase = open_cta(bars, NBAR, S_READ, OUT_FULL, reinterpret_cast<uint32_t*>(smem + kSmemBar + NBAR * 8), abort_flag);
  const uint32_t lead_bars = mapa_shared(smem_u32(bars), 0);
  auto wait = [&](int bar, uint32_t use, int site) {  // for phase `use` of a barrier
    return wait_for(&bars[bar], use & 1, abort_flag, p.status, site);
  };
  bool out_ok = steps == 0;

  if (steps > 0 && warp == 0) {
    if (lane == 0) {
      auto arm = [&](int bar, uint32_t bytes) {  // the bytes of both CTAs' loads, on the leader's barrier
        if (leader) mbar_expect_tx(&bars[bar], 2 * bytes);
        return lead_bars + bar * 8;
      };
      auto place = [&](int j, int& h, int& row) {
        h = hk * p.group + (first + j) / q_tiles;
        row = (first + j) % q_tiles * kTile;
      };
      int h, row;
      auto stats = [&](int j, uint32_t bar) {  // of this CTA's half of a tile's queries
        tma_load_2d_pair(&maps.stats, bar, smem + kSmemAux + (j % kLSlots) * kAuxBytes, 0,
                         (b * p.hq + h) * p.rows + row + static_cast<int>(rank) * 64);
      };
      const int ahead = min(steps, 2);
      uint32_t bar = arm(START, kTileBytes + ahead * (kHalfTile + kAuxBytes));
      load_resident(&maps.k[mi], bar, smem + kSmemK, row0, hk, bz);
      pdl_wait();  // the stats come from the launch before
      for (int j = 0; j < ahead; ++j) {
        place(j, h, row);
        load_rows(&maps.q[mi], bar, smem + smem_of(kQr, j), row, h, bz, rank);
        stats(j, bar);
      }
      bar = arm(S_READ, kTileBytes + kHalfTile);
      load_resident(&maps.v[mi], bar, smem + kSmemV, row0, hk, bz);
      for (int j = 0; j < ahead; ++j) {
        if (j > 0) bar = arm(S_READ + j, kHalfTile);
        place(j, h, row);
        load_rows(&maps.d_o[mi], bar, smem + smem_of(kOr, j), row, h, bz, rank);
      }
      int pd = 0, sr = ahead;  // steps whose loads on PD_READY / S_READ were issued
      for (int j = 0; j < steps; ++j) {
        if (!wait(S_FULL + (j & 1), j >> 1, kSiteProducer)) break;
        const bool more = j + 2 < steps;
        bar = arm(PD_READY + (j & 1), more ? 3 * kHalfTile + kAuxBytes : 2 * kHalfTile);
        ++pd;
        place(j, h, row);
        load_dims(&maps.d_o[mi], bar, smem + smem_of(kOd, j), row, h, bz, rank);
        load_dims(&maps.q[mi], bar, smem + smem_of(kQd, j), row, h, bz, rank);
        if (!more) continue;
        place(j + 2, h, row);
        stats(j + 2, bar);  // the slot's last readers, S and dP of step j - 2, are done: S(j) follows that step's gradients
        load_rows(&maps.q[mi], bar, smem + smem_of(kQr, j), row, h, bz, rank);
        if (!wait(DP_FULL + (j & 1), j >> 1, kSiteProducer)) break;
        bar = arm(S_READ + (j & 1), kHalfTile);
        ++sr;
        load_rows(&maps.d_o[mi], bar, smem + smem_of(kOr, j), row, h, bz, rank);
      }
      if (*abort_flag) {  // copies in flight: the last use of every barrier that counts bytes
        if (leader) {
          drain(&bars[START], 1, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteDrain);
          for (int s = 0; s < 2; ++s) {
            drain(&bars[PD_READY + s], (pd + 1 - s) / 2, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteDrain);
            drain(&bars[S_READ + s], (sr + 1 - s) / 2, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteDrain);
          }
        }
      }
    }
  } else if (steps > 0 && warp == 1) {
    if (leader && lane == 0) {  // X
      const uint64_t a = desc_k(smem + kSmemK), ones = desc_ones(smem + kSmemOnes);
      auto scores = [&](int j) {
        const uint32_t region = tbase + kColR + (j & 1) * 128;
        mma_f16_ss_pair(region, ones, desc_aux(smem + kSmemAux + (j % kLSlots) * kAuxBytes), kIdescScores, 0);
        issue_scores(region, a, desc_k(smem + smem_of(kQr, j)), true);
        tc_commit_pair(&bars[S_FULL + (j & 1)]);
      };
      bool ok = wait(START, 0, kSiteMma);
      if (ok) {
        tc_fence_after();
        scores(0);
        if (steps > 1) scores(1);
      }
      for (int j = 0; ok && j < steps; ++j) {
        if (!(ok = wait(PD_READY + (j & 1), j >> 1, kSiteMma))) break;
        tc_fence_after();
        const uint32_t region = tbase + kColR + (j & 1) * 128;
        issue_grad(tbase + kColDv, region, desc_mn(smem + smem_of(kOd, j)), j > 0);
        issue_grad(tbase + kColDk, region + kDs, desc_mn(smem + smem_of(kQd, j)), j > 0);
        if (j + 2 < steps) scores(j + 2);
      }
      tc_commit_pair(&bars[OUT_FULL]);
    }
  } else if (steps > 0 && warp == 2) {
    if (leader && lane == 0) {  // Y
      const uint64_t a = desc_k(smem + kSmemV), ones = desc_ones(smem + kSmemOnes + kOnesBytes);
      for (int j = 0; j < steps; ++j) {
        if (!wait(S_READ + (j & 1), j >> 1, kSiteMma)) break;
        tc_fence_after();
        const uint32_t region = tbase + kColR + (j & 1) * 128;
        issue_scores(region, a, desc_k(smem + smem_of(kOr, j)));
        // -delta comes last: dP is then what the rows' kernel summed, and where delta is that sum the two cancel exactly
        mma_f16_ss_pair(region, ones, desc_aux(smem + kSmemAux + (j % kLSlots) * kAuxBytes), kIdescScores, 1);
        tc_commit_pair(&bars[DP_FULL + (j & 1)]);
      }
    }
  } else if (steps > 0 && warp >= kControl) {
    const int wg = (warp - kControl) >> 2, quad = warp & 3;
    const uint32_t lane_col = tbase + (static_cast<uint32_t>(quad * 32) << 16) + kColR + kCols * wg;  // this warp's columns
    const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2);
    bool ok = true;
    for (int j = 0; j < steps && ok; ++j) {
      const uint32_t col = lane_col + (j & 1) * 128;
      if (!(ok = wait(S_FULL + (j & 1), j >> 1, kSiteScores))) break;
      tc_fence_after();
      float pr[kCols];
      uint32_t s[kCols], pk[kCols / 2];
      tmem_ld32(col, s);
      tmem_ld_wait(s);
      signal(lead_bars + (S_READ + (j & 1)) * 8);
#pragma unroll
      for (int i = 0; i < kCols; i += 2) {
        float x0, x1;
        f2_unpack(f2_mul(f2_pack(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), scale2), x0, x1);
        pr[i] = ex2_approx(x0);
        pr[i + 1] = ex2_approx(x1);
      }
      if (!(ok = wait(DP_FULL + (j & 1), j >> 1, kSiteScores))) break;
      tc_fence_after();
      tmem_ld32(col, s);
      tmem_ld_wait(s);
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) pk[i] = pack_bf16x2(pr[2 * i], pr[2 * i + 1]);
      tmem_st16(col, pk);
#pragma unroll
      for (int i = 0; i < kCols; i += 2) {
        float d0, d1;
        f2_unpack(f2_mul(f2_pack(pr[i], pr[i + 1]), f2_pack(__uint_as_float(s[i]), __uint_as_float(s[i + 1]))), d0, d1);
        pk[i / 2] = pack_bf16x2(d0, d1);
      }
      tmem_st16(col + kDs, pk);
      publish(lead_bars + (PD_READY + (j & 1)) * 8);
    }
    out_ok = ok && wait(OUT_FULL, 0, kSiteOut);
    tc_fence_after();
  }

  // The sums leave TMEM, the pair parts, and only then are the stores issued: parting waits for stores made before it.
  const int wg = (warp - kControl) >> 2, quad = warp & 3;
  const int row = row0 + quad * 32 + lane;
  uint32_t dv_sum[kCols], dk_sum[kCols];
  clear(dv_sum);
  clear(dk_sum);
  if (warp >= kControl && steps > 0 && out_ok) {
    const uint32_t col = tbase + (static_cast<uint32_t>(quad * 32) << 16) + kCols * wg;
    tmem_ld32(col + kColDv, dv_sum);
    tmem_ld_wait(dv_sum);
    tmem_ld32(col + kColDk, dk_sum);
    tmem_ld_wait(dk_sum);
    if (row >= kv_len) {  // rows behind the sequence are zero, whatever was summed there
      clear(dv_sum);
      clear(dk_sum);
    }
  }
  if (steps > 0) close_cta(tbase);
  if (warp >= kControl && out_ok && row < p.s_kv) {
    const bool parts = p.k_splits > 1;
    const long long at = (parts ? split * p.k_part : 0) +
                         ((static_cast<long long>(b) * p.s_kv + row) * p.hkv + hk) * kD + kCols * wg;
    store_share(dv_sum, 1.f, parts, p.dv, at);
    store_share(dk_sum, p.scale, parts, p.dk, at);
  }
}
}  // namespace dkdv

// ================================================================ dQ
namespace dq {
// Streamed operands of a key tile: K by rows (S), V by rows (dP), K by dims (dQ).
constexpr int kRegions = 3;  // score regions, and slots of K by rows and by dims
constexpr uint32_t kSmemQ = 0, kSmemO = kTileBytes, kSmemKr = 2 * kTileBytes;
constexpr uint32_t kSmemVr = kSmemKr + kRegions * kHalfTile, kSmemKd = kSmemVr + 2 * kHalfTile;
constexpr uint32_t kSmemBar = kSmemKd + kRegions * kHalfTile;
constexpr uint32_t kSmemBytes = kSmemBar + 256 + 1024;
// TMEM columns: three regions, each of a step's S, then dP, then dS; dQ.
constexpr uint32_t kColR = 0, kColDq = kRegions * 128;

// As in dkdv: X issues dQ(j), S(j+3), so S of step j complete frees the slots of dQ(j-3); Y issues dP(j).
enum Bar : int {
  START = 0,                    // Q and the first three tiles' K rows
  S_FULL = 1,                   // + step % 3
  DP_FULL = S_FULL + kRegions,  // + step % 2
  S_READ = DP_FULL + 2,         // Y's, + step % 2: S of step j is read; V's rows of j (and dO, for the first) are there
  DS_READY = S_READ + 2,        // X's, + step % 3: dS of step j; K's dims of j and K's rows of j + 3 are there
  Y_ISSUED = DS_READY + kRegions,  // + step % 2: dP of step j is queued on the tensor pipe
  OUT_FULL = Y_ISSUED + 2,
  NBAR = OUT_FULL + 1
};
static_assert(NBAR * 8 + 8 <= 256, "barriers, TMEM slot and abort flag fit their area");

template <int N>
VOMNI_DEV void body(const Maps<N>& maps, const Params& p, uint8_t* smem, int pair) {
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kSmemBar);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kSmemBar + NBAR * 8 + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair_row = pair % p.q_tiles2 * 2 * kTile;
  const int row0 = pair_row + static_cast<int>(rank) * kTile;  // this CTA's first query
  const int h = pair / p.q_tiles2 % p.hq, hk = h / p.group, z = pair / p.q_tiles2 / p.hq;
  const int seq = z / p.q_splits, split = z % p.q_splits;
  const int mi = N == 1 ? 0 : seq, bz = N == 1 ? seq : 0, b = p.b0 + seq;
  const int q_len = p.q_len[mi], kv_len = p.kv_len[mi];
  const int first = split * p.q_per;
  const int last = min(first + p.q_per, (kv_len + kTile - 1) / kTile);
  const int steps = pair_row < q_len ? max(last - first, 0) : 0;

  uint32_t tbase = 0;
  if (steps > 0)
    tbase = open_cta(bars, NBAR, S_READ, Y_ISSUED, reinterpret_cast<uint32_t*>(smem + kSmemBar + NBAR * 8), abort_flag);
  const uint32_t lead_bars = mapa_shared(smem_u32(bars), 0);
  auto wait = [&](int bar, uint32_t use, int site) {
    return site == kSiteScores ? mbar_poll(&bars[bar], use & 1, abort_flag, p.status, VOMNI_DEV_TIMEOUT_BASE + site)
                               : wait_for(&bars[bar], use & 1, abort_flag, p.status, site);
  };
  bool out_ok = steps == 0;

  if (steps > 0 && warp == 0) {
    if (lane == 0) {
      auto arm = [&](int bar, uint32_t bytes) {
        if (leader) mbar_expect_tx(&bars[bar], 2 * bytes);
        return lead_bars + bar * 8;
      };
      const int ahead = min(steps, kRegions), v_ahead = min(steps, 2);
      uint32_t bar = arm(START, kTileBytes + ahead * kHalfTile);
      load_resident(&maps.q[mi], bar, smem + kSmemQ, row0, h, bz);
      for (int j = 0; j < ahead; ++j)
        load_rows(&maps.k[mi], bar, smem + kSmemKr + j * kHalfTile, (first + j) * kTile, hk, bz, rank);
      bar = arm(S_READ, kTileBytes + kHalfTile);
      load_resident(&maps.d_o[mi], bar, smem + kSmemO, row0, h, bz);
      for (int j = 0; j < v_ahead; ++j) {
        if (j > 0) bar = arm(S_READ + j, kHalfTile);
        load_rows(&maps.v[mi], bar, smem + kSmemVr + j * kHalfTile, (first + j) * kTile, hk, bz, rank);
      }
      int ds = 0, sr = v_ahead;  // steps whose loads on DS_READY / S_READ were issued
      for (int j = 0; j < steps; ++j) {
        const int r = j % kRegions;
        if (!wait(S_FULL + r, j / kRegions, kSiteProducer)) break;
        const bool more = j + kRegions < steps;
        bar = arm(DS_READY + r, (more ? 2 : 1) * kHalfTile);
        ++ds;
        load_dims(&maps.k[mi], bar, smem + kSmemKd + r * kHalfTile, (first + j) * kTile, hk, bz, rank);
        if (more) load_rows(&maps.k[mi], bar, smem + kSmemKr + r * kHalfTile, (first + j + kRegions) * kTile, hk, bz, rank);
        if (j + 2 >= steps) continue;
        if (!wait(DP_FULL + (j & 1), j >> 1, kSiteProducer)) break;
        bar = arm(S_READ + (j & 1), kHalfTile);
        ++sr;
        load_rows(&maps.v[mi], bar, smem + kSmemVr + (j & 1) * kHalfTile, (first + j + 2) * kTile, hk, bz, rank);
      }
      if (*abort_flag && leader) {
        drain(&bars[START], 1, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteDrain);
        for (int s = 0; s < kRegions; ++s)
          drain(&bars[DS_READY + s], (ds + kRegions - 1 - s) / kRegions, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteDrain);
        for (int s = 0; s < 2; ++s)
          drain(&bars[S_READ + s], (sr + 1 - s) / 2, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteDrain);
      }
    }
  } else if (steps > 0 && warp == 1) {
    if (leader && lane == 0) {  // X
      const uint64_t a = desc_k(smem + kSmemQ);
      auto scores = [&](int r) {
        issue_scores(tbase + kColR + r * 128, a, desc_k(smem + kSmemKr + r * kHalfTile));
        tc_commit_pair(&bars[S_FULL + r]);
      };
      bool ok = wait(START, 0, kSiteMma);
      if (ok) {
        tc_fence_after();
        for (int j = 0; j < min(steps, kRegions); ++j) scores(j);
      }
      for (int j = 0, r = 0, use = 0; ok && j < steps; ++j) {
        if (!(ok = wait(DS_READY + r, use, kSiteMma))) break;
        tc_fence_after();
        issue_grad(tbase + kColDq, tbase + kColR + r * 128, desc_mn(smem + kSmemKd + r * kHalfTile), j > 0);
        // dP(j+1), which the score warps wait for next, goes ahead of S(j+3)
        if (j + 1 < steps && !(ok = wait(Y_ISSUED + ((j + 1) & 1), (j + 1) >> 1, kSiteMma))) break;
        if (j + kRegions < steps) scores(r);
        if (++r == kRegions) {
          r = 0;
          ++use;
        }
      }
      tc_commit_pair(&bars[OUT_FULL]);
    }
  } else if (steps > 0 && warp == 2) {
    if (leader && lane == 0) {  // Y
      const uint64_t a = desc_k(smem + kSmemO);
      for (int j = 0, r = 0; j < steps; ++j) {
        if (!wait(S_READ + (j & 1), j >> 1, kSiteMma)) break;
        tc_fence_after();
        issue_scores(tbase + kColR + r * 128, a, desc_k(smem + kSmemVr + (j & 1) * kHalfTile));
        tc_commit_pair(&bars[DP_FULL + (j & 1)]);
        mbar_arrive(&bars[Y_ISSUED + (j & 1)]);
        r = r + 1 == kRegions ? 0 : r + 1;
      }
    }
  } else if (steps > 0 && warp >= kControl) {
    const int wg = (warp - kControl) >> 2, quad = warp & 3;
    const uint32_t lane_col = tbase + (static_cast<uint32_t>(quad * 32) << 16) + kColR + kCols * wg;
    const int row = row0 + quad * 32 + lane;
    const long long at = (static_cast<long long>(b) * p.hq + h) * p.rows + row;
    const bool known = row < p.rows;  // the pair's second CTA may lie behind the last tile
    float nlse = -kNoKeys, neg_delta = 0.f;
    pdl_wait();  // the stats come from the launch before
    if (known) sum_stats(p.stats[at], p.scale_log2, nlse, neg_delta);
    const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2), nlse2 = f2_pack(nlse, nlse),
                   delta2 = f2_pack(neg_delta, neg_delta);
    bool ok = true;
    for (int j = 0, r = 0, use = 0; j < steps && ok; ++j) {
      const int valid = kv_len - (first + j) * kTile - kCols * wg;  // this warpgroup's columns that are keys
      const uint32_t col = lane_col + r * 128;
      if (!(ok = wait(S_FULL + r, use, kSiteScores))) break;
      tc_fence_after();
      float pr[kCols];
      uint32_t s[kCols], pk[kCols / 2];
      tmem_ld32(col, s);
      tmem_ld_wait(s);
      signal(lead_bars + (S_READ + (j & 1)) * 8);
#pragma unroll
      for (int i = 0; i < kCols; i += 2) {
        float x0, x1;
        f2_unpack(f2_fma(f2_pack(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), scale2, nlse2), x0, x1);
        pr[i] = ex2_approx(x0);
        pr[i + 1] = ex2_approx(x1);
      }
      if (valid < kCols) {  // columns behind the last key (zero scores) have no probability
#pragma unroll
        for (int i = 0; i < kCols; ++i) pr[i] = i < valid ? pr[i] : 0.f;
      }
      if (!(ok = wait(DP_FULL + (j & 1), j >> 1, kSiteScores))) break;
      tc_fence_after();
      tmem_ld32(col, s);
      tmem_ld_wait(s);
#pragma unroll
      for (int i = 0; i < kCols; i += 2) {
        float d0, d1;
        f2_unpack(f2_mul(f2_pack(pr[i], pr[i + 1]), f2_add(f2_pack(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), delta2)), d0, d1);
        pk[i / 2] = pack_bf16x2(d0, d1);
      }
      tmem_st16(col, pk);
      publish(lead_bars + (DS_READY + r) * 8);
      if (++r == kRegions) {
        r = 0;
        ++use;
      }
    }
    out_ok = ok && wait(OUT_FULL, 0, kSiteOut);
    tc_fence_after();
  }

  const int wg = (warp - kControl) >> 2, quad = warp & 3;
  const int row = row0 + quad * 32 + lane;
  uint32_t sum[kCols];
  clear(sum);
  if (warp >= kControl && steps > 0 && out_ok) {
    tmem_ld32(tbase + (static_cast<uint32_t>(quad * 32) << 16) + kColDq + kCols * wg, sum);
    tmem_ld_wait(sum);
    if (row >= q_len) clear(sum);
  }
  if (steps > 0) close_cta(tbase);
  if (warp >= kControl && out_ok && row < p.s_q) {
    const bool parts = p.q_splits > 1;
    const long long at = (parts ? split * p.q_part : 0) +
                         ((static_cast<long long>(b) * p.s_q + row) * p.hq + h) * kD + kCols * wg;
    store_share(sum, p.scale, parts, p.dq, at);
  }
}
}  // namespace dq

// A CTA pair of either kind: both are in one launch, so that the pairs of one fill the device while the other's last ones
// run.
constexpr uint32_t kSmemBytes = dkdv::kSmemBytes > dq::kSmemBytes ? dkdv::kSmemBytes : dq::kSmemBytes;
template <int N>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    attn_bwd_kernel(const __grid_constant__ Maps<N> maps, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int pair = blockIdx.x >> 1;
  if (pair < p.k_pairs)
    dkdv::body<N>(maps, p, smem, pair);
  else
    dq::body<N>(maps, p, smem, pair - p.k_pairs);
  pdl_wait();  // no CTA ends before the launch that it overlapped
}

// ================================================================ rows: lse and delta
// delta = dO O^T's diagonal, by the tensor cores in the order in which they sum dP's products: where a row of V is the
// row of O to the bit (a row with one key), dP - delta is exactly 0, as it should be, and so are dQ and dK. Summed by
// another order what is left of the two was rounding noise, all of the result (1e-7 of dP; 2 times fp32's own).
template <int N>
struct RowMaps {
  CUtensorMap o[N], d_o[N];  // as Maps
};
struct RowParams {
  const float* lse;   // [b, hq, 128, ceil(s_q / 128)]
  const float* dlse;  // the same, or null (0)
  int hq, rows, groups;
  int q_len[kMaxSeqs];
  int b0;
  float scale;
  uint4* stats;
  int* status;
};

// A CTA takes a tile of 128 rows of one head: dO's and O's, one 128 x 128 product of them, its diagonal, a thread a row.
// Rows behind a sequence's end (up to the tile's) get no probability. HBM-bound: 512 bytes a row; three CTAs an SM keep
// 192 KB of loads under way. 8190 x 40 rows 34 us, 4.9 TB/s (38 with plain loads and fused multiply-adds, four rows a half-warp);
// a single tile takes 2 us more than by those with a cold L2, the same with a warm one.
constexpr uint32_t kRowSmemBytes = 2 * kTileBytes + 1024;
constexpr uint32_t kIdescRows = idesc_bf16(128, 128, false);
template <int N>
__global__ void __launch_bounds__(128) attn_bwd_rows_kernel(const __grid_constant__ RowMaps<N> maps, const __grid_constant__ RowParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t bars[2];  // operands there, product done
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x % p.groups, h = blockIdx.x / p.groups % p.hq, seq = blockIdx.x / p.groups / p.hq, b = p.b0 + seq;
  const int mi = N == 1 ? 0 : seq, bz = N == 1 ? seq : 0;
  const int row0 = tile * kTile, row = row0 + static_cast<int>(threadIdx.x), len = p.q_len[mi];
  const bool any = row0 < len;
  if (any) {
    if (threadIdx.x == 0) {
      mbar_init(&bars[0], 1);
      mbar_init(&bars[1], 1);
      *abort_flag = 0;
      fence_mbar_init();
    }
    if (warp == 0) {
      tmem_alloc(&tmem_slot, kTile);
      tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  }
  pdl_trigger();  // not before this CTA has its TMEM: the dependents take all of an SM's
  const long long bh = static_cast<long long>(b) * p.hq + h;
  float l = p.scale > 0.f ? -kNoKeys : kNoKeys, delta = 0.f;
  if (any) {
    const long long at = (bh * 128 + threadIdx.x) * p.groups + tile;
    const float v = row < len ? p.lse[at] : 0.f, dlse = row < len && p.dlse ? p.dlse[at] : 0.f;
    if (threadIdx.x == 0) {
      const uint32_t bar = smem_u32(&bars[0]);
      mbar_expect_tx(&bars[0], 2 * kTileBytes);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        tma_load_4d(&maps.d_o[mi], bar, smem + i * kBox, (i >> 1) * 64, row0 + (i & 1) * 64, h, bz);
        tma_load_4d(&maps.o[mi], bar, smem + kTileBytes + i * kBox, (i >> 1) * 64, row0 + (i & 1) * 64, h, bz);
      }
      if (mbar_wait(&bars[0], 0, abort_flag, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteRows)) {
        tc_fence_after();
        const uint64_t x = desc_k(smem), y = desc_k(smem + kTileBytes);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint64_t off = ((kk >> 2) * 2 * kBox + (kk & 3) * 32) >> 4;
          mma_f16_ss(tmem_slot, x + off, y + off, kIdescRows, kk > 0);
        }
        tc_commit(&bars[1]);
      } else {
        drain(&bars[0], 1, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteDrain);
      }
    }
    const bool ok = mbar_wait(&bars[1], 0, abort_flag, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteRows);
    if (__all_sync(0xffffffffu, ok)) {
      tc_fence_after();
      uint32_t s[32];  // columns 32 warp ... of row threadIdx.x
      tmem_ld32(tmem_slot + (static_cast<uint32_t>(warp * 32) << 16) + warp * 32, s);
      tmem_ld_wait(s);
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (lane == i) delta = __uint_as_float(s[i]);
    }
    if (row < len) {
      if (isinf(v)) {
        delta = 0.f;  // no probabilities, whatever dlse holds
      } else {
        l = -v / p.scale;
        if (p.dlse) delta -= dlse;
      }
      if (fabsf(l) > kNoKeys) l = l > 0.f ? kNoKeys : -kNoKeys;
    } else {
      delta = 0.f;
    }
  }
  p.stats[bh * p.rows + row] = stats_of(l, -delta);
  if (any) {
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
      tc_fence_after();
      tmem_dealloc(tmem_slot, kTile);
    }
  }
}

// out = bf16(sum over parts), in order, of up to three gradients in one launch.
struct JoinParams {
  const float* parts[3];
  __nv_bfloat16* out[3];
  long long part[3];  // elements, 0 where there is nothing to join
  int n[3];
};
__global__ void __launch_bounds__(256) attn_bwd_join_kernel(const __grid_constant__ JoinParams p) {
  long long at = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) * 4;
  int t = 0;
  while (t < 3 && at >= p.part[t]) at -= p.part[t++];  // every part is a multiple of 128
  if (t == 3) return;
  const float* parts = p.parts[t] + at;
  float4 s = *reinterpret_cast<const float4*>(parts);
  for (int i = 1; i < p.n[t]; ++i) {
    const float4 u = *reinterpret_cast<const float4*>(parts + i * p.part[t]);
    s.x += u.x; s.y += u.y; s.z += u.z; s.w += u.w;
  }
  *reinterpret_cast<uint2*>(p.out[t] + at) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
}

// ================================================================ host
// How many CTA pairs share the walk of one dK/dV tile and of one dQ tile: the counts for which the launch is estimated to
// end first, in microseconds as measured at 1.7 GHz. A pair takes 1.5 us a step (dkdv) or 1.3 (dq) and 4 to start, fill and
// end; the pairs run on half as many slots as there are SMs, dK/dV first. Joining fp32 parts costs a launch and their
// traffic. 1 and 1 where the tiles alone fill the device (cross-attention of 8190 x 512 x 40 heads: 438 us with the 4
// dkdv splits of a rule that looked at that kind alone, 372 without).
constexpr int kMaxSplits = 16;
struct Work {
  long long k_outputs = 0, q_outputs = 0;  // tiles of 256 rows that have something to walk
  int k_walk = 0, q_walk = 0;              // steps of the longest walk
  long long k_steps = 0, q_steps = 0;      // of all walks
  double k_bytes = 0, q_bytes = 0;         // of one part of dk and dv, of dq
};
bool even_split(int tiles, int s, int& per) {
  per = (tiles + s - 1) / s;
  return (tiles + per - 1) / per == s;  // no empty splits
}
void choose_splits(const Work& w, int& k_splits, int& q_splits) {
  const double slots = num_sms() / 2 > 0 ? num_sms() / 2 : 1;
  k_splits = q_splits = 1;
  if (w.k_outputs + w.q_outputs > 16 * slots && w.k_outputs > slots) return;  // splits gain nothing there
  const double k_step = 1.5, q_step = 1.3, fixed = 4;
  double best = 0;
  for (int sk = 1; sk <= kMaxSplits && sk <= w.k_walk; ++sk) {
    int k_per, q_per;
    if (!even_split(w.k_walk, sk, k_per)) continue;
    for (int sq = 1; sq <= kMaxSplits && sq <= w.q_walk; ++sq) {
      if (!even_split(w.q_walk, sq, q_per)) continue;
      const double k_len = k_step * k_per + fixed, q_len = q_step * q_per + fixed;
      const double work = k_step * w.k_steps + q_step * w.q_steps + fixed * (w.k_outputs * sk + w.q_outputs * sq);
      double cost = std::max(work / slots + q_len / 2, std::max(k_len, q_len));
      if (sk > 1 || sq > 1) cost += 3 + 2e-6 / 6.5 * ((sk > 1 ? sk * w.k_bytes : 0) + (sq > 1 ? sq * w.q_bytes : 0));
      if (best == 0 || cost < best * 0.98) {
        best = cost;
        k_splits = sk;
        q_splits = sq;
      }
    }
  }
}

struct Plan {
  int rows;
  int q_splits, q_per, k_splits, k_per;  // splits of the dq walk (key tiles) and of the dkdv walk (query tiles)
  size_t row_bytes, q_bytes, k_bytes;    // stats; dq's parts; dk's parts, and dv's
  size_t bytes() const { return row_bytes + q_bytes + 2 * k_bytes; }
};
// q_lens, kv_lens: null for whole rows.
Plan plan_of(int b, int s_q, int s_kv, int hq, int hkv, const int* q_lens, const int* kv_lens) {
  Plan p;
  Work w;
  const int group = hq / hkv, n = q_lens || kv_lens ? b : 1, times = n == 1 ? b : 1;
  for (int i = 0; i < n; ++i) {
    const long long qt = ((q_lens ? q_lens[i] : s_q) + kTile - 1) / kTile, kt = ((kv_lens ? kv_lens[i] : s_kv) + kTile - 1) / kTile;
    if (qt == 0 || kt == 0) continue;
    const long long k_out = times * hkv * ((kt + 1) / 2), q_out = times * hq * ((qt + 1) / 2);
    w.k_outputs += k_out;
    w.q_outputs += q_out;
    w.k_steps += k_out * qt * group;
    w.q_steps += q_out * kt;
    w.k_walk = std::max<int>(w.k_walk, static_cast<int>(qt * group));
    w.q_walk = std::max<int>(w.q_walk, static_cast<int>(kt));
  }
  w.k_bytes = 8.0 * b * s_kv * hkv * kD;
  w.q_bytes = 4.0 * b * s_q * hq * kD;
  p.rows = (s_q + kTile - 1) / kTile * kTile;
  choose_splits(w, p.k_splits, p.q_splits);
  p.q_per = std::max(1, (w.q_walk + p.q_splits - 1) / p.q_splits);
  p.k_per = std::max(1, (w.k_walk + p.k_splits - 1) / p.k_splits);
  p.row_bytes = align_up(static_cast<size_t>(b) * hq * p.rows * sizeof(uint4), 256);
  p.q_bytes = p.q_splits > 1 ? static_cast<size_t>(p.q_splits) * b * s_q * hq * kD * 4 : 0;
  p.k_bytes = p.k_splits > 1 ? static_cast<size_t>(p.k_splits) * b * s_kv * hkv * kD * 4 : 0;
  return p;
}

bool bad_shape(int b, int s_q, int s_kv, int hq, int hkv, int d) {
  return d != kD || b <= 0 || s_q <= 0 || s_kv <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || hq > 65535 || b > 4095 ||
         s_q > (1 << 24) || s_kv > (1 << 24) ||
         static_cast<long long>(b) * hq * ((s_q + 127) / 128 * 128) > 0x7fffffffll;
}

// The maps of q, k, v, grad_o, o, in this order.
int make_maps(CUtensorMap* const (&maps)[5], const void* const (&base)[5], const long long (&st)[5][3], int batches, int q_len,
              int kv_len, int hq, int hkv) {
  for (int i = 0; i < 5; ++i) {
    const bool query = i == 0 || i > 2;
    const uint64_t dims[4] = {kD, static_cast<uint64_t>(query ? q_len : kv_len), static_cast<uint64_t>(query ? hq : hkv),
                              static_cast<uint64_t>(batches)};
    int rc = make_tmap_4d_bf16(maps[i], base[i], dims, st[i], 64, 64);
    if (rc) return rc;
  }
  return VOMNI_OK;
}

}  // namespace abwd
}  // namespace vomni

using namespace vomni;

static bool bad_lens(int b, int s_q, int s_kv, const int* q_lens, const int* kv_lens) {
  for (int i = 0; i < b; ++i)
    if ((q_lens && (q_lens[i] < 0 || q_lens[i] > s_q)) || (kv_lens && (kv_lens[i] < 0 || kv_lens[i] > s_kv))) return true;
  return false;
}

extern "C" size_t vomni_attention_bwd_workspace_bytes(int b, int s_q, int s_kv, int hq, int hkv, int d, const int* q_lens,
                                                      const int* kv_lens) {
  if (abwd::bad_shape(b, s_q, s_kv, hq, hkv, d) || bad_lens(b, s_q, s_kv, q_lens, kv_lens)) return 0;
  return abwd::plan_of(b, s_q, s_kv, hq, hkv, q_lens, kv_lens).bytes();
}

// Launches the rows' kernel and then the pairs, as its dependent, of batch elements [p.b0, p.b0 + n) with their maps.
template <int N>
static int launch_parts(const abwd::RowMaps<N>& row_maps, const abwd::RowParams& r, const abwd::Maps<N>& maps, abwd::Params p, int n,
                        cudaStream_t st) {
  using namespace abwd;
  const long long k_pairs = static_cast<long long>(p.k_tiles2) * p.hkv * n * p.k_splits;
  const long long pairs = k_pairs + static_cast<long long>(p.q_tiles2) * p.hq * n * p.q_splits;
  if (pairs > (1 << 30)) return VOMNI_EBADSHAPE;
  p.k_pairs = static_cast<int>(k_pairs);
  auto rows = attn_bwd_rows_kernel<N>;
  int rc = ensure_max_smem(rows, kRowSmemBytes);
  if (rc) return rc;
  rows<<<static_cast<unsigned>(n) * r.hq * r.groups, 128, kRowSmemBytes, st>>>(row_maps, r);  // at most 2^24 (bad_shape)
  VOMNI_CUDA_TRY(cudaGetLastError());
  auto kern = attn_bwd_kernel<N>;
  rc = ensure_max_smem(kern, kSmemBytes);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VOMNI_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, maps, p));
  return VOMNI_OK;
}

extern "C" int vomni_attention_bwd_lse(const void* grad_o, const float* grad_lse, const void* q, const void* k, const void* v,
                                       const void* o, const float* lse, int b, int s_q, int s_kv, int hq, int hkv, int d,
                                       const long long* strides, const int* q_lens, const int* kv_lens, float softmax_scale,
                                       void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                                       vomni_stream_t stream) {
  using namespace abwd;
  if (!grad_o || !q || !k || !v || !o || !lse || !strides || !dq || !dk || !dv || !workspace) return VOMNI_EINVAL;
  if (!(std::fabs(softmax_scale) >= 1e-20f && std::fabs(softmax_scale) <= 1e20f)) return VOMNI_EINVAL;
  if (bad_shape(b, s_q, s_kv, hq, hkv, d)) return VOMNI_EBADSHAPE;
  if (bad_lens(b, s_q, s_kv, q_lens, kv_lens)) return VOMNI_EBADSHAPE;
  const uintptr_t al = reinterpret_cast<uintptr_t>(grad_o) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                       reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(dq) |
                       reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv) |
                       reinterpret_cast<uintptr_t>(workspace);
  if (al & 15) return VOMNI_EALIGN;
  if ((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(grad_lse)) & 3) return VOMNI_EALIGN;
  const Plan plan = plan_of(b, s_q, s_kv, hq, hkv, q_lens, kv_lens);
  if (workspace_bytes < plan.bytes()) return VOMNI_EWORKSPACE;
  // strides: (row, head, batch) of q, k, v, grad_o, o in elements, multiples of 8 where the extent is over 1
  long long st5[5][3];
  for (int t = 0; t < 5; ++t) {
    const int ext[3] = {t == 1 || t == 2 ? s_kv : s_q, t == 1 || t == 2 ? hkv : hq, b};
    for (int i = 0; i < 3; ++i) {
      const long long e = strides[t * 3 + i];
      if (ext[i] > 1 && (e <= 0 || e % 8 || e > (1ll << 38))) return VOMNI_EALIGN;
      st5[t][i] = ext[i] > 1 ? e : 0;
    }
  }
  int rc = require_sm100();
  if (rc) return rc;
  rc = bind_context(reinterpret_cast<const void*>(abwd::attn_bwd_join_kernel));
  if (rc) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool lens = q_lens || kv_lens;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Params p = {};
  p.s_q = s_q;
  p.s_kv = s_kv;
  p.hq = hq;
  p.hkv = hkv;
  p.group = hq / hkv;
  p.rows = plan.rows;
  p.stats = reinterpret_cast<const uint4*>(ws);
  p.scale = softmax_scale;
  p.scale_log2 = softmax_scale * kLog2e;
  p.status = device_status_ptr();
  p.k_tiles2 = (s_kv + 2 * kTile - 1) / (2 * kTile);
  p.q_tiles2 = (s_q + 2 * kTile - 1) / (2 * kTile);
  p.k_splits = plan.k_splits;
  p.k_per = plan.k_per;
  p.q_splits = plan.q_splits;
  p.q_per = plan.q_per;
  p.q_part = static_cast<long long>(b) * s_q * hq * kD;
  p.k_part = static_cast<long long>(b) * s_kv * hkv * kD;
  uint8_t* parts = ws + plan.row_bytes;
  p.dq = plan.q_splits > 1 ? parts : dq;
  p.dk = plan.k_splits > 1 ? parts + plan.q_bytes : dk;
  p.dv = plan.k_splits > 1 ? parts + plan.q_bytes + plan.k_bytes : dv;

  const int chunk = lens ? kMaxSeqs : b;
  auto fill_lens = [&](int b0, int n) {
    p.b0 = b0;
    for (int i = 0; i < (lens ? n : 1); ++i) {
      p.q_len[i] = q_lens ? q_lens[b0 + i] : s_q;
      p.kv_len[i] = kv_lens ? kv_lens[b0 + i] : s_kv;
    }
  };
  for (int b0 = 0; b0 < b; b0 += chunk) {
    const int n = std::min(chunk, b - b0);
    fill_lens(b0, n);
    RowParams r = {};
    r.lse = lse;
    r.dlse = grad_lse;
    r.hq = hq;
    r.rows = plan.rows;
    r.groups = plan.rows / kTile;
    for (int i = 0; i < kMaxSeqs; ++i) r.q_len[i] = p.q_len[i];
    r.b0 = b0;
    r.scale = softmax_scale;
    r.stats = const_cast<uint4*>(p.stats);
    r.status = p.status;
    CUtensorMap stats_map;
    rc = make_tmap_2d_plain(&stats_map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, ws, 8, static_cast<uint64_t>(b) * hq * plan.rows, 16,
                            8, 64);
    if (rc) return rc;
    const __nv_bfloat16* all[5] = {static_cast<const __nv_bfloat16*>(q), static_cast<const __nv_bfloat16*>(k),
                                   static_cast<const __nv_bfloat16*>(v), static_cast<const __nv_bfloat16*>(grad_o),
                                   static_cast<const __nv_bfloat16*>(o)};
    if (!lens) {
      Maps<1> maps;
      RowMaps<1> row_maps;
      maps.stats = stats_map;
      const void* const base[5] = {all[0], all[1], all[2], all[3], all[4]};
      rc = make_maps({maps.q, maps.k, maps.v, maps.d_o, row_maps.o}, base, st5, b, s_q, s_kv, hq, hkv);
      row_maps.d_o[0] = maps.d_o[0];
      if (!rc) rc = launch_parts<1>(row_maps, r, maps, p, n, st);
    } else {
      Maps<kMaxSeqs> maps;
      RowMaps<kMaxSeqs> row_maps;
      maps.stats = stats_map;
      for (int i = 0; i < n && !rc; ++i) {
        const void* base[5];
        for (int t = 0; t < 5; ++t) base[t] = all[t] + (b0 + i) * st5[t][2];
        // a length of 0 is never loaded from, but a map has no empty extent
        rc = make_maps({&maps.q[i], &maps.k[i], &maps.v[i], &maps.d_o[i], &row_maps.o[i]},
                       {base[0], base[1], base[2], base[3], base[4]}, st5, 1, std::max(p.q_len[i], 1), std::max(p.kv_len[i], 1), hq, hkv);
        row_maps.d_o[i] = maps.d_o[i];
      }
      if (!rc) rc = launch_parts<kMaxSeqs>(row_maps, r, maps, p, n, st);
    }
    if (rc) return rc;
  }
  if (plan.q_splits > 1 || plan.k_splits > 1) {
    JoinParams j = {};
    const void* from[3] = {p.dq, p.dk, p.dv};
    void* to[3] = {dq, dk, dv};
    for (int t = 0; t < 3; ++t) {
      j.parts[t] = static_cast<const float*>(from[t]);
      j.out[t] = static_cast<__nv_bfloat16*>(to[t]);
      j.n[t] = t ? plan.k_splits : plan.q_splits;
      j.part[t] = j.n[t] > 1 ? (t ? p.k_part : p.q_part) : 0;
    }
    const long long blocks = ((j.part[0] + j.part[1] + j.part[2]) / 4 + 255) / 256;
    if (blocks > 0x7fffffffll) return VOMNI_EBADSHAPE;
    attn_bwd_join_kernel<<<static_cast<unsigned>(blocks), 256, 0, st>>>(j);
    VOMNI_CUDA_TRY(cudaGetLastError());
  }
  return VOMNI_OK;
}

extern "C" int vomni_attention_bwd(const void* grad_o, const void* q, const void* k, const void* v, const void* o,
                                   const float* lse, int b, int s_q, int s_kv, int hq, int hkv, int d,
                                   const long long* strides, const int* q_lens, const int* kv_lens, float softmax_scale,
                                   void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                                   vomni_stream_t stream) {
  return vomni_attention_bwd_lse(grad_o, nullptr, q, k, v, o, lse, b, s_q, s_kv, hq, hkv, d, strides, q_lens, kv_lens,
                                 softmax_scale, dq, dk, dv, workspace, workspace_bytes, stream);
}
