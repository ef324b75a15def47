// Attention's backward pass for sm_100a, which recomputes the probabilities from the forward's log-sum-exp:
//     P = exp(scale Q K^T - lse)            dV = P^T dO
//     dS = P (dO V^T - delta)               delta = rowsum(dO O)
//     dQ = scale dS K                       dK = scale dS^T Q
// The forward's lse is the one of ring_attention_const_max_fwd(training=True)
// (vllm_omni_neuron/kernels/nkilib/experimental/attention/ring_attention_const_max_fwd.py:1062-1065), so the gradients
// of a part of the keys are those of that part of the whole softmax, and parts add up.
//
// Two tensor-core kernels, one per side of the score matrix, so that every gradient is summed in one CTA pair's TMEM
// in a fixed order and written once: no atomics, no fp32 gradient in HBM, the same bits every time. The price is
// that S and dP are formed twice: 7 matrix products instead of the 5 of one pass that adds dQ with atomics.
//   dkdv: a pair of CTAs holds 256 keys of one key head (128 rows of TMEM in each) and walks the query tiles of every
//         query head that shares it: S^T = K Q^T, dP^T = V dO^T, then dV += P^T dO and dK += dS^T Q with P^T, dS^T
//         read straight from TMEM.
//   dq:   a pair holds 256 queries of one head and walks the key tiles: S = Q K^T, dP = dO V^T, dQ += dS K.
// Both use tcgen05 cta_group::2 (M = 256, N = 128): each CTA stages half of every streamed operand, split by rows for
// the S and dP products and by head dimension for the others, as a one-CTA M = 128 product would need 128 B of
// shared-memory operands a clock and leave no room for the loads.
// Warps: 0 TMA producer, 1 MMA issuer (the even CTA's), 2..9 exponentials and gradients of the scores: a thread owns
// one TMEM lane (a key in dkdv, a query in dq), warpgroup wg the columns [64 wg, 64 wg + 64).
// Matrix products per 128 x 128 scores of a CTA: 512 clocks each; exponentials: 1024 clocks of the MUFU unit.
//
// Rounding: P and dS are rounded to bf16 as tensor-core operands (2^-8 relative each, at most); everything else is fp32 until the
// gradients are rounded once.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "common.cuh"
#include "host_util.h"

namespace vomni {
namespace abwd {

constexpr int kD = 128;
constexpr int kTile = 128;              // columns of a step (queries in dkdv, keys in dq); rows of a CTA
constexpr int kThreads = 64 + 256;
constexpr int kMaxSeqs = 16;            // batch elements of a launch with lengths of their own
constexpr uint32_t kBox = 64 * 64 * 2;  // 8 KB: one TMA box, 64 rows x 64 dims, 128-byte swizzled
constexpr uint32_t kTileBytes = 4 * kBox;  // resident operand: [2 dim halves][2 row halves] boxes
constexpr uint32_t kHalfTile = 2 * kBox;   // a CTA's half of a streamed operand
constexpr float kNoKeys = 1e30f;        // log2-sum-exp of a row without keys: its probabilities are 0
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kScoreWarps = 16;    // score warps of both CTAs: arrivals per READY phase

// One set of maps for a batch of equal lengths (the batch element is a coordinate), or one per batch element
// whose extents end at its lengths: rows behind them read as zero, whatever they hold.
template <int N>
struct Maps {
  CUtensorMap q[N], k[N], v[N], d_o[N];
};

struct Params {
  int b0;                     // first batch element of this launch
  int s_q, s_kv, hq, hkv, group;
  int q_len[kMaxSeqs], kv_len[kMaxSeqs];  // of each batch element (of the launch); [0] for all in a uniform one
  int rows;                   // row pitch of lse2 / delta: s_q rounded up to whole tiles
  const float* lse2;          // [b * hq, rows]: log2(e) * lse, kNoKeys behind the last query
  const float* delta;         // [b * hq, rows], 0 behind the last query
  float scale, scale_log2;
  int splits, per_split;      // the walked tiles are dealt to splits of per_split tiles
  void* out0;                 // dq | dk: bf16 [b, s, heads, 128], or fp32 parts [split][b, s, heads, 128]
  void* out1;                 // dv
  long long part;             // elements of one part
  int* status;
};

// P / dS in TMEM: the bf16 values of columns [16 kk, 16 kk + 16) sit in the 8 TMEM columns from pcol(kk). Each
// warpgroup writes over the score columns that it has read itself (wg 0: columns 0-63, wg 1: 64-127).
__host__ __device__ constexpr uint32_t pcol(int kk) { return kk * 8 + (kk >= 4 ? 32 : 0); }

constexpr uint32_t kIdescScores = idesc_bf16(256, 128, false);
constexpr uint32_t kIdescGrad = idesc_bf16(256, 128, true);

// scores[256 x 128] = A (resident, 128 rows in each CTA) B^T (streamed, 64 rows in each CTA), both K-major over d.
VOMNI_DEV void issue_scores(uint32_t d, uint64_t a, uint64_t b) {
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
    mma_f16_ss_pair(d, a + (((kk >> 2) * 2 * kBox + (kk & 3) * 32) >> 4), b + (((kk >> 2) * kBox + (kk & 3) * 32) >> 4),
                    kIdescScores, kk > 0);
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

// This warp's columns are in TMEM (its stores completed): one arrival on the leader's barrier.
VOMNI_DEV void publish(uint32_t bar_cluster) {
  tmem_st_wait();
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive_cluster(bar_cluster);
}

// 64 columns of one row of a gradient, times `scale`, to the output row (bf16, or fp32 parts). `computed`: the columns
// hold sums (uniform over the CTA); rows that are not in the sequence (`in`) are written as zero, `ok`: in the tensor.
VOMNI_DEV void store_half_row(uint32_t col, float scale, bool computed, bool in, bool ok, bool parts, void* out,
                              long long at) {
#pragma unroll 1
  for (int ch = 0; ch < 2; ++ch) {
    uint32_t o[32];
    if (computed) {
      tmem_ld32(col + ch * 32, o);
      tmem_ld_wait(o);
    }
    if (!ok) continue;
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = computed && in ? __uint_as_float(o[i]) * scale : 0.f;
    if (parts) {
      float4* dst = reinterpret_cast<float4*>(static_cast<float*>(out) + at + ch * 32);
#pragma unroll
      for (int i = 0; i < 8; ++i) dst[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
      uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(out) + at + ch * 32);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        dst[i] = make_uint4(pack_bf16x2(v[8 * i], v[8 * i + 1]), pack_bf16x2(v[8 * i + 2], v[8 * i + 3]),
                            pack_bf16x2(v[8 * i + 4], v[8 * i + 5]), pack_bf16x2(v[8 * i + 6], v[8 * i + 7]));
    }
  }
}

// A CTA that gave up waits (bounded) for the copies it may still have in flight: barrier `bar` has had `uses` loads.
VOMNI_DEV void drain(uint64_t* bar, int uses, int* status, int code) {
  if (uses <= 0) return;
  int ignored = 0;
  mbar_wait(bar, (uses - 1) & 1, &ignored, status, code);
}

// Device status sites (VOMNI_DEV_TIMEOUT_BASE + site).
enum Site : int { kSiteProducer = 0x40, kSiteMma = 0x41, kSiteScores = 0x42, kSiteOut = 0x43, kSiteDrain = 0x44 };

// ================================================================ dK, dV
namespace dkdv {
// Streamed operands of a query tile, two slots each: Q and dO by rows (for S^T, dP^T), dO and Q by dims (for dV, dK).
constexpr uint32_t kSmemK = 0, kSmemV = kTileBytes, kSmemStream = 2 * kTileBytes;
constexpr int kSlots = 2, kLSlots = 4;
constexpr uint32_t kSlotBytes = kHalfTile;  // 16 KB
constexpr uint32_t smem_of(int kind, int slot) { return kSmemStream + (kind * kSlots + slot) * kSlotBytes; }
constexpr int kQr = 0, kOr = 1, kOd = 2, kQd = 3;
constexpr uint32_t kSmemL = kSmemStream + 4 * kSlots * kSlotBytes;  // [kLSlots][lse2 128 | delta 128] fp32
constexpr uint32_t kSmemBar = kSmemL + kLSlots * 1024;
constexpr uint32_t kSmemBytes = kSmemBar + 256 + 1024;
// TMEM columns: S^T / P^T, dP^T / dS^T, dV, dK.
constexpr uint32_t kColS = 0, kColDp = 128, kColDv = 256, kColDk = 384;

// Slot-indexed barriers complete once every kSlots steps. S_FULL + s and DP_FULL + s also tell the producers which
// slots are free: MMAs complete in issue order, so S of step j + 1 complete means dV of step j complete, and dP of
// step j + 1 means dK of step j. Each is waited for before the load that its next phase depends on, so no
// wait can miss a phase.
enum Bar : int {
  KV_FULL = 0,
  FULL = 1,                        // + kind * kSlots + slot
  L_FULL = FULL + 4 * kSlots,      // + step % kLSlots, this CTA's own
  S_FULL = L_FULL + kLSlots,       // + step % 2
  DP_FULL = S_FULL + 2,            // + step % 2
  P_READY = DP_FULL + 2,
  DS_READY = P_READY + 1,
  OUT_FULL = DS_READY + 1,
  NBAR = OUT_FULL + 1
};
static_assert(NBAR * 8 + 8 <= 256, "barriers, TMEM slot and abort flag fit their area");

template <int N>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    attn_bwd_dkdv_kernel(const __grid_constant__ Maps<N> maps, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kSmemBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kSmemBar + NBAR * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kSmemBar + NBAR * 8 + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair_row = (blockIdx.x >> 1) * 2 * kTile;
  const int row0 = pair_row + static_cast<int>(rank) * kTile;  // this CTA's first key
  const int hk = blockIdx.y;
  const int seq = blockIdx.z / p.splits, split = blockIdx.z % p.splits;
  const int mi = N == 1 ? 0 : seq, bz = N == 1 ? seq : 0, b = p.b0 + seq;
  const int q_len = p.q_len[mi], kv_len = p.kv_len[mi];
  const int q_tiles = (q_len + kTile - 1) / kTile;
  // this split's steps of the walk over (query head of the group, query tile)
  const int first = split * p.per_split;
  const int last = min(first + p.per_split, q_tiles * p.group);
  const int steps = pair_row < kv_len ? max(last - first, 0) : 0;

  if (steps > 0) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < NBAR; ++i) mbar_init(&bars[i], i == P_READY || i == DS_READY ? kScoreWarps : 1);
      *abort_flag = 0;
      fence_mbar_init();
    }
    if (warp == 1) {
      tmem_alloc_pair(tmem_slot, 512);
      tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
  }
  const uint32_t tbase = steps > 0 ? *tmem_slot : 0;
  const uint32_t lead_bars = mapa_shared(smem_u32(bars), 0);
  bool out_ok = steps == 0;

  if (steps > 0 && warp == 0) {
    if (lane == 0) {
      const uint32_t kv_bar = lead_bars + KV_FULL * 8;
      if (leader) mbar_expect_tx(&bars[KV_FULL], 4 * kTileBytes);
      load_resident(&maps.k[mi], kv_bar, smem + kSmemK, row0, hk, bz);
      load_resident(&maps.v[mi], kv_bar, smem + kSmemV, row0, hk, bz);
      int issued[4] = {};  // loads of each kind
      bool ok = true;
      for (int j = 0; j < steps && ok; ++j) {
        const int s = j & 1, t = first + j;
        const int h = hk * p.group + t / q_tiles, row = (t % q_tiles) * kTile;
        const uint32_t full = lead_bars + (FULL + s) * 8;
        auto arm = [&](int kind) {
          if (leader) mbar_expect_tx(&bars[FULL + kind * kSlots + s], 2 * kSlotBytes);
          ++issued[kind];
          return full + kind * kSlots * 8;
        };
        auto wait = [&](int bar, int step) {
          return mbar_wait_spin(&bars[bar + (step & 1)], (step >> 1) & 1, abort_flag, p.status,
                                VOMNI_DEV_TIMEOUT_BASE + kSiteProducer);
        };
        // lse2 and delta of the step (slot's last reader: step j - 4, long done once dP of step j - 2 is)
        if (j >= kSlots && !(ok = wait(S_FULL, j - 2))) break;
        uint32_t bar = arm(kQr);
        load_rows(&maps.q[mi], bar, smem + smem_of(kQr, s), row, h, bz, rank);
        if (j >= kSlots && !(ok = wait(DP_FULL, j - 2))) break;
        bar = arm(kOr);
        load_rows(&maps.d_o[mi], bar, smem + smem_of(kOr, s), row, h, bz, rank);
        const int l = j % kLSlots;
        const long long at = (static_cast<long long>(b) * p.hq + h) * p.rows + row;
        mbar_expect_tx(&bars[L_FULL + l], 1024);
        bulk_g2s(smem + kSmemL + l * 1024, p.lse2 + at, 512, &bars[L_FULL + l]);
        bulk_g2s(smem + kSmemL + l * 1024 + 512, p.delta + at, 512, &bars[L_FULL + l]);
        if (j >= kSlots && !(ok = wait(S_FULL, j - 1))) break;
        bar = arm(kOd);
        load_dims(&maps.d_o[mi], bar, smem + smem_of(kOd, s), row, h, bz, rank);
        if (j >= kSlots && !(ok = wait(DP_FULL, j - 1))) break;
        bar = arm(kQd);
        load_dims(&maps.q[mi], bar, smem + smem_of(kQd, s), row, h, bz, rank);
      }
      if (*abort_flag) {
        if (leader) {
          drain(&bars[KV_FULL], 1, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteDrain);
          for (int kind = 0; kind < 4; ++kind)
            for (int s = 0; s < kSlots; ++s)
              drain(&bars[FULL + kind * kSlots + s], (issued[kind] + kSlots - 1 - s) / kSlots, p.status,
                    VOMNI_DEV_TIMEOUT_BASE + kSiteDrain);
        }
        for (int l = 0; l < kLSlots; ++l)
          drain(&bars[L_FULL + l], (issued[kOr] + kLSlots - 1 - l) / kLSlots, p.status,
                VOMNI_DEV_TIMEOUT_BASE + kSiteDrain);
      }
    }
  } else if (steps > 0 && warp == 1) {
    // Order per step j: dV(j), S(j+1) over P(j), dK(j), dP(j+1) over dS(j): while one of P and dS is formed, the
    // tensor pipe works on the other.
    if (leader && lane == 0) {
      const uint64_t dk_a = desc_k(smem + kSmemK), dv_a = desc_k(smem + kSmemV);
      auto wait = [&](int bar, uint32_t parity) {
        return mbar_wait_spin(&bars[bar], parity, abort_flag, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteMma);
      };
      auto full = [&](int kind, int j) { return wait(FULL + kind * kSlots + (j & 1), (j >> 1) & 1); };
      auto scores = [&](int j) {
        if (!full(kQr, j)) return false;
        tc_fence_after();
        issue_scores(tbase + kColS, dk_a, desc_k(smem + smem_of(kQr, j & 1)));
        tc_commit_pair(&bars[S_FULL + (j & 1)]);
        return true;
      };
      auto dprobs = [&](int j) {
        if (!full(kOr, j)) return false;
        tc_fence_after();
        issue_scores(tbase + kColDp, dv_a, desc_k(smem + smem_of(kOr, j & 1)));
        tc_commit_pair(&bars[DP_FULL + (j & 1)]);
        return true;
      };
      bool ok = wait(KV_FULL, 0) && scores(0) && dprobs(0);
      for (int j = 0; ok && j < steps; ++j) {
        if (!(ok = wait(P_READY, j & 1) && full(kOd, j))) break;
        tc_fence_after();
        issue_grad(tbase + kColDv, tbase + kColS, desc_mn(smem + smem_of(kOd, j & 1)), j > 0);
        if (j + 1 < steps && !(ok = scores(j + 1))) break;
        if (!(ok = wait(DS_READY, j & 1) && full(kQd, j))) break;
        tc_fence_after();
        issue_grad(tbase + kColDk, tbase + kColDp, desc_mn(smem + smem_of(kQd, j & 1)), j > 0);
        if (j + 1 < steps && !(ok = dprobs(j + 1))) break;
      }
      tc_commit_pair(&bars[OUT_FULL]);
    }
  } else if (steps > 0) {
    const int wg = (warp - 2) >> 2, quad = warp & 3;
    const uint32_t lane_addr = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t col_s = tbase + lane_addr + kColS, col_dp = tbase + lane_addr + kColDp;
    const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2);
    auto wait = [&](int bar, uint32_t parity) {
      return mbar_wait_spin(&bars[bar], parity, abort_flag, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteScores);
    };
    bool ok = true;
    for (int j = 0; j < steps && ok; ++j) {
      const float* lse2 = reinterpret_cast<const float*>(smem + kSmemL + (j % kLSlots) * 1024) + 64 * wg;
      const float* delta = lse2 + 128;
      if (!(ok = wait(L_FULL + j % kLSlots, (j / kLSlots) & 1) && wait(S_FULL + (j & 1), (j >> 1) & 1))) break;
      tc_fence_after();
      float pr[64];
#pragma unroll
      for (int ch = 0; ch < 2; ++ch) {
        uint32_t s[32], pk[16];
        tmem_ld32(col_s + 64 * wg + 32 * ch, s);
        tmem_ld_wait(s);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 l = *reinterpret_cast<const float2*>(lse2 + 32 * ch + 2 * i);
          float x0, x1;
          f2_unpack(f2_fma(f2_pack(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale2, f2_pack(-l.x, -l.y)),
                    x0, x1);
          pr[32 * ch + 2 * i] = ex2_approx(x0);
          pr[32 * ch + 2 * i + 1] = ex2_approx(x1);
          pk[i] = pack_bf16x2(pr[32 * ch + 2 * i], pr[32 * ch + 2 * i + 1]);
        }
        tmem_st16(col_s + pcol(4 * wg + 2 * ch), pk);
      }
      publish(lead_bars + P_READY * 8);
      if (!(ok = wait(DP_FULL + (j & 1), (j >> 1) & 1))) break;
      tc_fence_after();
#pragma unroll
      for (int ch = 0; ch < 2; ++ch) {
        uint32_t s[32], pk[16];
        tmem_ld32(col_dp + 64 * wg + 32 * ch, s);
        tmem_ld_wait(s);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 d = *reinterpret_cast<const float2*>(delta + 32 * ch + 2 * i);
          const int c = 32 * ch + 2 * i;
          pk[i] = pack_bf16x2(pr[c] * (__uint_as_float(s[2 * i]) - d.x), pr[c + 1] * (__uint_as_float(s[2 * i + 1]) - d.y));
        }
        tmem_st16(col_dp + pcol(4 * wg + 2 * ch), pk);
      }
      publish(lead_bars + DS_READY * 8);
    }
    out_ok = ok && mbar_wait_spin(&bars[OUT_FULL], 0, abort_flag, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteOut);
    tc_fence_after();
  }

  if (warp >= 2 && out_ok) {
    const int wg = (warp - 2) >> 2, quad = warp & 3;
    const uint32_t lane_addr = static_cast<uint32_t>(quad * 32) << 16;
    const int row = row0 + quad * 32 + lane;
    const bool parts = p.splits > 1;
    const long long at = (parts ? split * p.part : 0) +
                         ((static_cast<long long>(b) * p.s_kv + row) * p.hkv + hk) * kD + 64 * wg;
    store_half_row(tbase + lane_addr + kColDv + 64 * wg, 1.f, steps > 0, row < kv_len, row < p.s_kv, parts, p.out1, at);
    store_half_row(tbase + lane_addr + kColDk + 64 * wg, p.scale, steps > 0, row < kv_len, row < p.s_kv, parts, p.out0, at);
  }
  if (steps > 0) {
    tc_fence_before();
    cluster_sync();
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc_pair(tbase, 512);
    }
  }
}
}  // namespace dkdv

// ================================================================ dQ
namespace dq {
// A stage: K and V by rows (S, dP) and K by dims (dQ).
constexpr int kStages = 3;
constexpr uint32_t kStageBytes = 3 * kHalfTile;
constexpr uint32_t kSmemQ = 0, kSmemO = kTileBytes, kSmemStage = 2 * kTileBytes;
constexpr uint32_t kSmemBar = kSmemStage + kStages * kStageBytes;
constexpr uint32_t kSmemBytes = kSmemBar + 256 + 1024;
constexpr uint32_t kKr = 0, kVr = kHalfTile, kKd = 2 * kHalfTile;
// TMEM columns: S of even and odd steps, dP / dS, dQ.
constexpr uint32_t kColS = 0, kColDp = 256, kColDq = 384;

enum Bar : int {
  Q_FULL = 0,
  FULL = 1,
  EMPTY = FULL + kStages,
  S_FULL = EMPTY + kStages,  // + step % 2
  DP_FULL = S_FULL + 2,
  DS_READY = DP_FULL + 1,
  OUT_FULL = DS_READY + 1,
  NBAR = OUT_FULL + 1
};
static_assert(NBAR * 8 + 8 <= 256, "barriers, TMEM slot and abort flag fit their area");

template <int N>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    attn_bwd_dq_kernel(const __grid_constant__ Maps<N> maps, const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kSmemBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kSmemBar + NBAR * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kSmemBar + NBAR * 8 + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair_row = (blockIdx.x >> 1) * 2 * kTile;
  const int row0 = pair_row + static_cast<int>(rank) * kTile;  // this CTA's first query
  const int h = blockIdx.y, hk = h / p.group;
  const int seq = blockIdx.z / p.splits, split = blockIdx.z % p.splits;
  const int mi = N == 1 ? 0 : seq, bz = N == 1 ? seq : 0, b = p.b0 + seq;
  const int q_len = p.q_len[mi], kv_len = p.kv_len[mi];
  const int first = split * p.per_split;
  const int last = min(first + p.per_split, (kv_len + kTile - 1) / kTile);
  const int steps = pair_row < q_len ? max(last - first, 0) : 0;

  if (steps > 0) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < NBAR; ++i) mbar_init(&bars[i], i == DS_READY ? kScoreWarps : 1);
      *abort_flag = 0;
      fence_mbar_init();
    }
    if (warp == 1) {
      tmem_alloc_pair(tmem_slot, 512);
      tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
  }
  const uint32_t tbase = steps > 0 ? *tmem_slot : 0;
  const uint32_t lead_bars = mapa_shared(smem_u32(bars), 0);
  bool out_ok = steps == 0;

  if (steps > 0 && warp == 0) {
    if (lane == 0) {
      const uint32_t q_bar = lead_bars + Q_FULL * 8;
      if (leader) mbar_expect_tx(&bars[Q_FULL], 4 * kTileBytes);
      load_resident(&maps.q[mi], q_bar, smem + kSmemQ, row0, h, bz);
      load_resident(&maps.d_o[mi], q_bar, smem + kSmemO, row0, h, bz);
      int done = 0;
      for (int j = 0; j < steps; ++j, ++done) {
        const int st = j % kStages, use = j / kStages;
        if (use > 0 && !mbar_wait_spin(&bars[EMPTY + st], (use - 1) & 1, abort_flag, p.status,
                                       VOMNI_DEV_TIMEOUT_BASE + kSiteProducer))
          break;
        const uint32_t bar = lead_bars + (FULL + st) * 8;
        uint8_t* dst = smem + kSmemStage + st * kStageBytes;
        const int row = (first + j) * kTile;
        if (leader) mbar_expect_tx(&bars[FULL + st], 2 * kStageBytes);
        load_rows(&maps.k[mi], bar, dst + kKr, row, hk, bz, rank);
        load_rows(&maps.v[mi], bar, dst + kVr, row, hk, bz, rank);
        load_dims(&maps.k[mi], bar, dst + kKd, row, hk, bz, rank);
      }
      if (*abort_flag && leader) {
        drain(&bars[Q_FULL], 1, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteDrain);
        for (int s = 0; s < kStages; ++s)
          drain(&bars[FULL + s], (done + kStages - 1 - s) / kStages, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteDrain);
      }
    }
  } else if (steps > 0 && warp == 1) {
    // Order per step j: dQ(j), dP(j+1) over dS(j), S(j+2) over S(j): the scores run two steps ahead, so that the
    // exponentials of step j + 1 overlap dQ(j) and dP(j+1), and its dS overlaps S(j+2).
    if (leader && lane == 0) {
      const uint64_t q_a = desc_k(smem + kSmemQ), o_a = desc_k(smem + kSmemO);
      auto wait = [&](int bar, uint32_t parity) {
        return mbar_wait_spin(&bars[bar], parity, abort_flag, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteMma);
      };
      auto stage = [&](int j) { return smem + kSmemStage + (j % kStages) * kStageBytes; };
      auto scores = [&](int j) {  // the first use of its stage
        if (!wait(FULL + j % kStages, (j / kStages) & 1)) return false;
        tc_fence_after();
        issue_scores(tbase + kColS + (j & 1) * 128, q_a, desc_k(stage(j) + kKr));
        tc_commit_pair(&bars[S_FULL + (j & 1)]);
        return true;
      };
      auto dprobs = [&](int j) {
        issue_scores(tbase + kColDp, o_a, desc_k(stage(j) + kVr));
        tc_commit_pair(&bars[DP_FULL]);
      };
      bool ok = wait(Q_FULL, 0) && scores(0);
      if (ok) dprobs(0);
      if (ok && steps > 1) ok = scores(1);
      for (int j = 0; ok && j < steps; ++j) {
        if (!(ok = wait(DS_READY, j & 1))) break;
        tc_fence_after();
        issue_grad(tbase + kColDq, tbase + kColDp, desc_mn(stage(j) + kKd), j > 0);
        tc_commit_pair(&bars[EMPTY + j % kStages]);
        if (j + 1 < steps) dprobs(j + 1);
        if (j + 2 < steps && !(ok = scores(j + 2))) break;
      }
      tc_commit_pair(&bars[OUT_FULL]);
    }
  } else if (steps > 0) {
    const int wg = (warp - 2) >> 2, quad = warp & 3;
    const uint32_t lane_addr = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t col_dp = tbase + lane_addr + kColDp;
    const int row = row0 + quad * 32 + lane;
    const long long at = (static_cast<long long>(b) * p.hq + h) * p.rows + row;
    const bool known = row < p.rows;  // the pair's second CTA may lie behind the last tile
    const float nlse = known ? -p.lse2[at] : -kNoKeys, delta = known ? p.delta[at] : 0.f;
    const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2), nlse2 = f2_pack(nlse, nlse);
    auto wait = [&](int bar, uint32_t parity) {
      return mbar_wait_spin(&bars[bar], parity, abort_flag, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteScores);
    };
    bool ok = true;
    for (int j = 0; j < steps && ok; ++j) {
      const int valid = kv_len - (first + j) * kTile - 64 * wg;  // this warpgroup's columns that are keys
      if (!(ok = wait(S_FULL + (j & 1), (j >> 1) & 1))) break;
      tc_fence_after();
      float pr[64];
#pragma unroll
      for (int ch = 0; ch < 2; ++ch) {
        uint32_t s[32];
        tmem_ld32(tbase + lane_addr + kColS + (j & 1) * 128 + 64 * wg + 32 * ch, s);
        tmem_ld_wait(s);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float x0, x1;
          f2_unpack(f2_fma(f2_pack(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale2, nlse2), x0, x1);
          pr[32 * ch + 2 * i] = ex2_approx(x0);
          pr[32 * ch + 2 * i + 1] = ex2_approx(x1);
        }
      }
      if (valid < 64) {  // columns behind the last key (zero scores) have no probability
#pragma unroll
        for (int i = 0; i < 64; ++i) pr[i] = i < valid ? pr[i] : 0.f;
      }
      if (!(ok = wait(DP_FULL, j & 1))) break;
      tc_fence_after();
#pragma unroll
      for (int ch = 0; ch < 2; ++ch) {
        uint32_t s[32], pk[16];
        tmem_ld32(col_dp + 64 * wg + 32 * ch, s);
        tmem_ld_wait(s);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int c = 32 * ch + 2 * i;
          pk[i] = pack_bf16x2(pr[c] * (__uint_as_float(s[2 * i]) - delta), pr[c + 1] * (__uint_as_float(s[2 * i + 1]) - delta));
        }
        tmem_st16(col_dp + pcol(4 * wg + 2 * ch), pk);
      }
      publish(lead_bars + DS_READY * 8);
    }
    out_ok = ok && mbar_wait_spin(&bars[OUT_FULL], 0, abort_flag, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteOut);
    tc_fence_after();
  }

  if (warp >= 2 && out_ok) {
    const int wg = (warp - 2) >> 2, quad = warp & 3;
    const int row = row0 + quad * 32 + lane;
    const bool parts = p.splits > 1;
    const long long at = (parts ? split * p.part : 0) +
                         ((static_cast<long long>(b) * p.s_q + row) * p.hq + h) * kD + 64 * wg;
    store_half_row(tbase + (static_cast<uint32_t>(quad * 32) << 16) + kColDq + 64 * wg, p.scale, steps > 0,
                   row < q_len, row < p.s_q, parts, p.out0, at);
  }
  if (steps > 0) {
    tc_fence_before();
    cluster_sync();
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc_pair(tbase, 512);
    }
  }
}
}  // namespace dq

// ================================================================ rows: delta and lse2
struct RowParams {
  const __nv_bfloat16* o;
  const __nv_bfloat16* d_o;
  const float* lse;  // [b, hq, 128, ceil(s_q / 128)]
  long long o_s, o_h, o_b, do_s, do_h, do_b;  // strides in elements
  int b, hq, s_q, rows, groups;
  int lens;  // q_len per batch element (b <= kMaxSeqs), else q_len[0]
  int q_len[kMaxSeqs];
  int b0;
  float* lse2;
  float* delta;
};

// One half-warp per row, 8 values a lane. Rows behind a sequence's end (up to the tile's) get no probability.
__global__ void __launch_bounds__(256) attn_bwd_rows_kernel(const __grid_constant__ RowParams p) {
  const long long n = static_cast<long long>(p.b) * p.hq * p.rows;
  const long long i = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 4;
  if (i >= n) return;  // n is a multiple of 128: whole warps leave
  const int sub = threadIdx.x & 15;
  const int row = static_cast<int>(i % p.rows);
  const int h = static_cast<int>(i / p.rows % p.hq), seq = static_cast<int>(i / p.rows / p.hq), b = p.b0 + seq;
  const bool in = row < (p.lens ? p.q_len[seq] : p.q_len[0]);
  float acc = 0.f;
  if (in) {
    const uint4 x = *reinterpret_cast<const uint4*>(p.o + b * p.o_b + h * p.o_h + row * p.o_s + sub * 8);
    const uint4 y = *reinterpret_cast<const uint4*>(p.d_o + b * p.do_b + h * p.do_h + row * p.do_s + sub * 8);
    const __nv_bfloat162* a = reinterpret_cast<const __nv_bfloat162*>(&x);
    const __nv_bfloat162* c = reinterpret_cast<const __nv_bfloat162*>(&y);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = __bfloat1622float2(a[k]), g = __bfloat1622float2(c[k]);
      acc = fmaf(f.x, g.x, fmaf(f.y, g.y, acc));
    }
  }
#pragma unroll
  for (int s = 8; s > 0; s >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, s);
  if (sub == 0) {
    const long long bh = static_cast<long long>(b) * p.hq + h;
    float l = kNoKeys;
    if (in) {
      const float v = p.lse[(bh * 128 + (row & 127)) * p.groups + (row >> 7)];
      l = v == -INFINITY ? kNoKeys : v * kLog2e;
    }
    p.lse2[bh * p.rows + row] = l;
    p.delta[bh * p.rows + row] = acc;
  }
}

// out = bf16(sum over parts), in order.
__global__ void __launch_bounds__(256) attn_bwd_join_kernel(const float* __restrict__ parts, int n_parts, long long part,
                                                            __nv_bfloat16* __restrict__ out) {
  const long long at = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) * 4;
  if (at >= part) return;  // part is a multiple of 128
  float4 s = *reinterpret_cast<const float4*>(parts + at);
  for (int i = 1; i < n_parts; ++i) {
    const float4 t = *reinterpret_cast<const float4*>(parts + i * part + at);
    s.x += t.x; s.y += t.y; s.z += t.z; s.w += t.w;
  }
  *reinterpret_cast<uint2*>(out + at) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
}

// ================================================================ host
// How many CTA pairs share one output tile's walk of `tiles` steps: the count whose waves of pairs take the
// least time, a pair costing its steps and about two more to start and finish (and half a step more to write
// and join fp32 parts). 1 where the output tiles alone fill the device.
int choose_splits(long long outputs, int tiles) {
  const long long slots = num_sms() / 2 > 0 ? num_sms() / 2 : 1;
  int best = 1;
  double best_cost = 0;
  for (int s = 1; s <= 16 && s <= tiles; ++s) {
    const int per = (tiles + s - 1) / s;
    if ((tiles + per - 1) / per != s) continue;  // no empty splits
    const double cost = static_cast<double>((outputs * s + slots - 1) / slots) * (per + 2 + (s > 1 ? 1 : 0));
    if (s == 1 || cost < best_cost * 0.97) {
      best = s;
      best_cost = cost;
    }
  }
  return best;
}

struct Plan {
  int rows;
  int q_splits, q_per, k_splits, k_per;  // splits of the dq walk (key tiles) and of the dkdv walk (query tiles)
  size_t row_bytes, part_bytes;
};
Plan plan_of(int b, int s_q, int s_kv, int hq, int hkv) {
  Plan p;
  const int q_tiles = (s_q + kTile - 1) / kTile, k_tiles = (s_kv + kTile - 1) / kTile;
  p.rows = q_tiles * kTile;
  p.q_splits = choose_splits(static_cast<long long>(b) * hq * ((q_tiles + 1) / 2), k_tiles);
  p.q_per = (k_tiles + p.q_splits - 1) / p.q_splits;
  const int walk = q_tiles * (hq / hkv);
  p.k_splits = choose_splits(static_cast<long long>(b) * hkv * ((k_tiles + 1) / 2), walk);
  p.k_per = (walk + p.k_splits - 1) / p.k_splits;
  p.row_bytes = align_up(static_cast<size_t>(b) * hq * p.rows * sizeof(float), 256);
  const size_t dq = p.q_splits > 1 ? static_cast<size_t>(p.q_splits) * b * s_q * hq * kD * 4 : 0;
  const size_t dkv = p.k_splits > 1 ? 2 * static_cast<size_t>(p.k_splits) * b * s_kv * hkv * kD * 4 : 0;
  p.part_bytes = std::max(dq, dkv);  // the two kernels' parts live one after the other
  return p;
}

bool bad_shape(int b, int s_q, int s_kv, int hq, int hkv, int d) {
  return d != kD || b <= 0 || s_q <= 0 || s_kv <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || hq > 65535 || b > 4095 ||
         s_q > (1 << 24) || s_kv > (1 << 24) || static_cast<long long>((s_q + 127) / 128) * (hq / hkv) > (1 << 30);
}

int make_maps(CUtensorMap* q, CUtensorMap* k, CUtensorMap* v, CUtensorMap* o, const void* const (&base)[4],
              const long long (&st)[4][3], int batches, int q_len, int kv_len, int hq, int hkv) {
  CUtensorMap* maps[4] = {q, k, v, o};
  for (int i = 0; i < 4; ++i) {
    const bool query = i == 0 || i == 3;
    const uint64_t dims[4] = {kD, static_cast<uint64_t>(query ? q_len : kv_len), static_cast<uint64_t>(query ? hq : hkv),
                              static_cast<uint64_t>(batches)};
    int rc = make_tmap_4d_bf16(maps[i], base[i], dims, st[i], 64, 64);
    if (rc) return rc;
  }
  return VOMNI_OK;
}

int join(const void* parts, int n, long long part, void* out, cudaStream_t st) {
  const long long blocks = (part / 4 + 255) / 256;
  if (blocks > 0x7fffffffll) return VOMNI_EBADSHAPE;
  attn_bwd_join_kernel<<<static_cast<unsigned>(blocks), 256, 0, st>>>(static_cast<const float*>(parts), n, part,
                                                                      static_cast<__nv_bfloat16*>(out));
  VOMNI_CUDA_TRY(cudaGetLastError());
  return VOMNI_OK;
}

}  // namespace abwd
}  // namespace vomni

using namespace vomni;

extern "C" size_t vomni_attention_bwd_workspace_bytes(int b, int s_q, int s_kv, int hq, int hkv, int d) {
  if (abwd::bad_shape(b, s_q, s_kv, hq, hkv, d)) return 0;
  const abwd::Plan p = abwd::plan_of(b, s_q, s_kv, hq, hkv);
  return 2 * p.row_bytes + p.part_bytes;
}

// Launches both kernels for batch elements [p.b0, p.b0 + n) with their maps.
template <int N>
static int launch_pair(const abwd::Maps<N>& maps, abwd::Params p, const abwd::Plan& plan, int n, int dq_or_dkdv,
                       cudaStream_t st) {
  using namespace abwd;
  if (dq_or_dkdv == 0) {
    auto kern = dkdv::attn_bwd_dkdv_kernel<N>;
    int rc = ensure_max_smem(kern, dkdv::kSmemBytes);
    if (rc) return rc;
    kern<<<dim3(2 * ((p.s_kv + 255) / 256), p.hkv, n * p.splits), kThreads, dkdv::kSmemBytes, st>>>(maps, p);
  } else {
    auto kern = dq::attn_bwd_dq_kernel<N>;
    int rc = ensure_max_smem(kern, dq::kSmemBytes);
    if (rc) return rc;
    kern<<<dim3(2 * ((p.s_q + 255) / 256), p.hq, n * p.splits), kThreads, dq::kSmemBytes, st>>>(maps, p);
  }
  VOMNI_CUDA_TRY(cudaGetLastError());
  return VOMNI_OK;
}

extern "C" int vomni_attention_bwd(const void* grad_o, const void* q, const void* k, const void* v, const void* o,
                                   const float* lse, int b, int s_q, int s_kv, int hq, int hkv, int d,
                                   const long long* strides, const int* q_lens, const int* kv_lens, float softmax_scale,
                                   void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes,
                                   vomni_stream_t stream) {
  using namespace abwd;
  if (!grad_o || !q || !k || !v || !o || !lse || !strides || !dq || !dk || !dv || !workspace) return VOMNI_EINVAL;
  if (bad_shape(b, s_q, s_kv, hq, hkv, d)) return VOMNI_EBADSHAPE;
  for (int i = 0; i < b; ++i)
    if ((q_lens && (q_lens[i] < 0 || q_lens[i] > s_q)) || (kv_lens && (kv_lens[i] < 0 || kv_lens[i] > s_kv)))
      return VOMNI_EBADSHAPE;
  const uintptr_t al = reinterpret_cast<uintptr_t>(grad_o) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                       reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(dq) |
                       reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv) |
                       reinterpret_cast<uintptr_t>(workspace);
  if (al & 15) return VOMNI_EALIGN;
  if (reinterpret_cast<uintptr_t>(lse) & 3) return VOMNI_EALIGN;
  const Plan plan = plan_of(b, s_q, s_kv, hq, hkv);
  if (workspace_bytes < 2 * plan.row_bytes + plan.part_bytes) return VOMNI_EWORKSPACE;
  // strides: (row, head, batch) of q, k, v, grad_o, o in elements, multiples of 8 where the extent is over 1
  long long st4[4][3], so[3];
  for (int t = 0; t < 5; ++t) {
    const int ext[3] = {t == 1 || t == 2 ? s_kv : s_q, t == 1 || t == 2 ? hkv : hq, b};
    for (int i = 0; i < 3; ++i) {
      const long long e = strides[t * 3 + i];
      if (ext[i] > 1 && (e <= 0 || e % 8 || e > (1ll << 38))) return VOMNI_EALIGN;
      (t < 4 ? st4[t][i] : so[i]) = ext[i] > 1 ? e : 0;
    }
  }
  int rc = require_sm100();
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
  p.lse2 = reinterpret_cast<float*>(ws);
  p.delta = reinterpret_cast<float*>(ws + plan.row_bytes);
  p.scale = softmax_scale;
  p.scale_log2 = softmax_scale * kLog2e;
  p.status = device_status_ptr();
  void* parts = ws + 2 * plan.row_bytes;

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
    r.o = static_cast<const __nv_bfloat16*>(o);
    r.d_o = static_cast<const __nv_bfloat16*>(grad_o);
    r.lse = lse;
    r.o_s = so[0]; r.o_h = so[1]; r.o_b = so[2];
    r.do_s = st4[3][0]; r.do_h = st4[3][1]; r.do_b = st4[3][2];
    r.b = n;
    r.hq = hq;
    r.s_q = s_q;
    r.rows = plan.rows;
    r.groups = (s_q + 127) / 128;
    r.lens = lens;
    for (int i = 0; i < kMaxSeqs; ++i) r.q_len[i] = p.q_len[i];
    r.b0 = b0;
    r.lse2 = const_cast<float*>(p.lse2);
    r.delta = const_cast<float*>(p.delta);
    const long long blocks = (static_cast<long long>(n) * hq * plan.rows * 16 + 255) / 256;
    if (blocks > 0x7fffffffll) return VOMNI_EBADSHAPE;
    attn_bwd_rows_kernel<<<static_cast<unsigned>(blocks), 256, 0, st>>>(r);
    VOMNI_CUDA_TRY(cudaGetLastError());
  }
  for (int pass = 0; pass < 2; ++pass) {  // dK and dV, then dQ
    p.splits = pass == 0 ? plan.k_splits : plan.q_splits;
    p.per_split = pass == 0 ? plan.k_per : plan.q_per;
    p.part = static_cast<long long>(b) * (pass == 0 ? s_kv : s_q) * (pass == 0 ? hkv : hq) * kD;
    const bool split = p.splits > 1;
    p.out0 = split ? parts : pass == 0 ? dk : dq;
    p.out1 = pass == 0 ? (split ? static_cast<float*>(parts) + p.splits * p.part : dv) : nullptr;
    for (int b0 = 0; b0 < b; b0 += chunk) {
      const int n = std::min(chunk, b - b0);
      if (static_cast<long long>(n) * p.splits > 65535) return VOMNI_EBADSHAPE;
      fill_lens(b0, n);
      if (!lens) {
        Maps<1> maps;
        const void* const base[4] = {q, k, v, grad_o};
        rc = make_maps(maps.q, maps.k, maps.v, maps.d_o, base, st4, b, s_q, s_kv, hq, hkv);
        if (rc) return rc;
        rc = launch_pair<1>(maps, p, plan, n, pass, st);
      } else {
        Maps<kMaxSeqs> maps;
        for (int i = 0; i < n; ++i) {
          const void* base[4];
          const void* all[4] = {q, k, v, grad_o};
          for (int t = 0; t < 4; ++t) base[t] = static_cast<const __nv_bfloat16*>(all[t]) + (b0 + i) * st4[t][2];
          const void* const fixed[4] = {base[0], base[1], base[2], base[3]};
          // a length of 0 is never loaded from, but a map has no empty extent
          rc = make_maps(&maps.q[i], &maps.k[i], &maps.v[i], &maps.d_o[i], fixed, st4, 1, std::max(p.q_len[i], 1),
                         std::max(p.kv_len[i], 1), hq, hkv);
          if (rc) return rc;
        }
        rc = launch_pair<kMaxSeqs>(maps, p, plan, n, pass, st);
      }
      if (rc) return rc;
    }
    if (split) {
      rc = join(parts, p.splits, p.part, pass == 0 ? dk : dq, st);
      if (rc) return rc;
      if (pass == 0 && (rc = join(p.out1, p.splits, p.part, dv, st))) return rc;
    }
  }
  return VOMNI_OK;
}
