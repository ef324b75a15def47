// The norms before and after a block, fused with its gate and residual scale, and their gradients:
//     y   = post(x) * post_w                     post: LayerNorm | RMSNorm | none
//     r   = residual + gate * y                  (residual_out = bf16(r))
//     n   = norm(r),  out = n * mul + add        norm: the same three
// The statistics and out come from the unrounded fp32 r; each result is rounded to bf16 once. Without x
// the branch is absent (r = residual) and only the norm is left.
//
// Gradients, from x, the stored bf16 r and the gradients dr', dout of residual_out and out:
//     g  = dout * mul,  dr = dr' + s_r (g - [mean g] - n mean(g n))          [..]: LayerNorm only
//     h  = dr * gate * post_w,  dx = s_x (h - [mean h] - y mean(h y)),  dresidual = dr
//     dgate = sum dr y post_w,  dpost_w = sum dr gate y,  dmul = sum dout n,  dadd = sum dout
// with n and y the normalised rows and s their 1 / deviation, recomputed here: the forward pass keeps
// nothing but r. The column sums need three accumulators per column, A = sum dr y, M = sum dout n and
// D = sum dout, per modulation row: gate and post_w are constant in the sum, so
// dgate = post_w A and dpost_w = sum over modulation rows of gate A.
//
// HBM-bound: 4 rows of 2H bytes a token forward, 6 backward, each read or written once. The rows come a few at a
// time through a ring in shared memory; a thread owns chunks of 8 adjacent columns of all of them. The kernels are persistent, so
// that in the backward pass a thread's column sums stay in its registers over all rows of its CTA; the CTAs' sums
// go to a workspace and are added in a fixed order by a second kernel (no atomics: the same call gives the same bits).
// Measured over several GPUs, 32760 x 5120: forward 224 to 236 us (0.87 to 0.91 of the measured copy rate), backward 354 to 382 us (0.80
// to 0.87).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"
#include "host_util.h"

namespace vomni {
namespace sandwich {

constexpr int kMaxH = 8192;  // 512 threads of two chunks
constexpr int kLayer = 0, kNone = 2, kAsked = 3;  // 1: RMSNorm
constexpr size_t kSmemPerSm = 200 * 1024;
constexpr int kPerGate = 1, kPerMul = 2, kPerAdd = 4;

struct Params {
  const __nv_bfloat16* x;         // sub-layer output [rows, H] or null
  const __nv_bfloat16* residual;  // forward: the stream before; backward: the stored residual_out
  const __nv_bfloat16* d_res;     // backward: gradient of residual_out or null
  const __nv_bfloat16* d_out;     // backward: gradient of out or null
  const float* gate;              // [n_mod or 1, H] or null (1)
  const float* post_w;            // [H] or null (1)
  const float* mul;               // [n_mod or 1, H] or null (1)
  const float* add;               // [n_mod or 1, H] or null (0)
  long long rows_per_mod;
  long long gate_step, mul_step, add_step;  // H where per modulation row, else 0
  int H, post, norm;
  float eps, inv_h;
  __nv_bfloat16* out0;  // forward: residual_out; backward: dx
  __nv_bfloat16* out1;  // forward: out; backward: dresidual
  float* parts;         // backward: [n_mod][lanes][3][H]
  int* status;          // device status word (bounded-wait timeouts)
  int slots;            // ring slots
};
constexpr int kBuf = 8 * 32;  // up to eight sums of 32 warps

VOMNI_DEV void load8(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// ---------------------------------------------------------------- sums over a row
// Sums N values over a warp with N - 1 + log2(32 / N) shuffles: halves of the lanes exchange halves of the values until
// each group of 32 / N lanes holds one value. Returns the sum of value lane / (32 / N).
template <int N>
VOMNI_DEV float warp_fold(float (&v)[N]) {
  const int lane = threadIdx.x & 31;
  int width = 16;
#pragma unroll
  for (int n = N; n > 1; n /= 2, width /= 2) {
    const bool upper = lane & width;
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      const float send = upper ? v[i] : v[i + n / 2], keep = upper ? v[i + n / 2] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, width);
    }
  }
#pragma unroll
  for (; width > 0; width /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], width);
  return v[0];
}

// Sums N values over the threads that share a row (or a few rows): kLanes lanes of a warp, or (0) the whole CTA through
// shared memory. Every thread ends with the same sums, added in an order that only the CTA's size sets. `turn`
// alternates between two buffers: a buffer is written again only after a barrier that follows its last read. Entries
// of warps that the CTA does not have are zero from the start. Returns whether any thread said `bad` (kVote).
template <int N, int kLanes, bool kVote = false>
VOMNI_DEV bool row_sum(float (&v)[N], float (*buf)[kBuf], int& turn, bool bad = false) {
  if constexpr (kLanes > 0) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int o = kLanes / 2; o > 0; o /= 2) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    return bad;
  }
  constexpr int kGroup = 32 / N;
  const int lane = threadIdx.x & 31;
  float s = warp_fold<N>(v);
  float* b = buf[turn];
  turn ^= 1;
  if (lane % kGroup == 0) b[lane / kGroup * 32 + (threadIdx.x >> 5)] = s;
  if (kVote)
    bad = __syncthreads_or(bad);
  else
    __syncthreads();
  b += lane * N;  // value lane / kGroup, N of its 32 warps
  if constexpr (N == 8) {
    const float4 x = reinterpret_cast<const float4*>(b)[0], y = reinterpret_cast<const float4*>(b)[1];
    s = ((x.x + x.y) + (x.z + x.w)) + ((y.x + y.y) + (y.z + y.w));
  } else if constexpr (N == 4) {
    const float4 x = *reinterpret_cast<const float4*>(b);
    s = (x.x + x.y) + (x.z + x.w);
  } else if constexpr (N == 2) {
    const float2 x = *reinterpret_cast<const float2*>(b);
    s = x.x + x.y;
  } else {
    s = b[0];
  }
#pragma unroll
  for (int o = kGroup / 2; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xffffffffu, s, i * kGroup);
  return bad;
}

// The values of R rows that a thread owns (C of each) as fp32 pairs: the packed arithmetic halves the instructions,
// which bound the backward pass before it (87 a value, 64 % of the issue slots at half the present speed).
template <int R, int C>
struct Vals {
  uint64_t v[R][C / 2];
};
VOMNI_DEV uint64_t both(float x) { return f2_pack(x, x); }
VOMNI_DEV float halves_sum(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}

template <int NV>
VOMNI_DEV void centre(uint64_t (&v)[NV * 4], float mean, const bool (&in)[NV]) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const uint64_t neg = both(in[j] ? -mean : 0.f);
#pragma unroll
    for (int i = 4 * j; i < 4 * j + 4; ++i) v[i] = f2_add(v[i], neg);
  }
}

// x -> its normalised values. Two passes (mean, then squared deviations) in fp32. Columns behind
// the row's end (whole chunks: in[j] false) hold zeros before and after.
template <int R, int C, int kLanes>
VOMNI_DEV void normalise(Vals<R, C>& x, int kind, const bool (&in)[C / 8], const Params& p, float (*buf)[kBuf],
                         int& turn) {
  if (kind == kNone) return;
  float s[R];
  if (kind == kLayer) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      uint64_t t = x.v[r][0];
#pragma unroll
      for (int i = 1; i < C / 2; ++i) t = f2_add(t, x.v[r][i]);
      s[r] = halves_sum(t);
    }
    row_sum<R, kLanes>(s, buf, turn);
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int j = 0; j < C / 8; ++j) {
        const uint64_t neg = both(in[j] ? -s[r] * p.inv_h : 0.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[r][4 * j + i] = f2_add(x.v[r][4 * j + i], neg);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    uint64_t t = f2_mul(x.v[r][0], x.v[r][0]);
#pragma unroll
    for (int i = 1; i < C / 2; ++i) t = f2_fma(x.v[r][i], x.v[r][i], t);
    s[r] = halves_sum(t);
  }
  row_sum<R, kLanes>(s, buf, turn);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint64_t rstd = both(rsqrtf(s[r] * p.inv_h + p.eps));
#pragma unroll
    for (int i = 0; i < C / 2; ++i) x.v[r][i] = f2_mul(x.v[r][i], rstd);
  }
}

// ---------------------------------------------------------------- rows in shared memory
// A CTA's rows come R at a time (adjacent rows: one bulk copy per tensor) through a ring of `slots` slots; one thread
// issues the copies, slots - 1 groups ahead.
constexpr int kMaxSlots = 4;
constexpr int kSiteRowWait = 0x18, kSiteRowDrain = 0x19;

struct Ring {
  uint4* mem;  // [slots][tensors][R * H / 8]
  uint64_t* full;
  int slots, tensors, chunks;  // chunks: R * H / 8
};

template <int R>
VOMNI_DEV void ring_issue(const Ring& g, const __nv_bfloat16* const (&src)[4], long long row, long long end, int H, int slot) {
  if (row >= end) return;
  const uint32_t bytes = static_cast<uint32_t>(min(static_cast<long long>(R), end - row)) * H * 2u;
  mbar_expect_tx(&g.full[slot], bytes * g.tensors);
  uint4* dst = g.mem + static_cast<size_t>(slot) * g.tensors * g.chunks;
#pragma unroll
  for (int t = 0, n = 0; t < 4; ++t)
    if (src[t]) bulk_g2s(dst + (n++) * g.chunks, src[t] + row * H, bytes, &g.full[slot]);
}

// The walk of a CTA over its groups of R rows of one modulation row: groups lane, lane + lanes, ... of
// ceil(rows_per_mod / R). body(row, rows, slot base) runs between the wait for the group and the barrier that frees
// its slot.
template <int R, typename Body>
VOMNI_DEV void walk_rows(const Params& p, const __nv_bfloat16* const (&src)[4], int tensors, uint8_t* smem, uint64_t* full,
                         int* abort_flag, Body&& body) {
  Ring g{reinterpret_cast<uint4*>(smem), full, p.slots, tensors, R * p.H / 8};
  volatile int* abort = abort_flag;
  if (threadIdx.x == 0) {
    for (int s = 0; s < g.slots; ++s) mbar_init(&full[s], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  const long long begin = static_cast<long long>(blockIdx.y) * p.rows_per_mod, end = begin + p.rows_per_mod;
  const long long first = begin + static_cast<long long>(blockIdx.x) * R, step = static_cast<long long>(gridDim.x) * R;
  long long ahead = first;
  if (threadIdx.x == 0)
    for (int s = 0; s < g.slots - 1; ++s, ahead += step) ring_issue<R>(g, src, ahead, end, p.H, s);
  int slot = 0;
  uint32_t phase = 0;
  long long row = first;
  for (; row < end; row += step) {
    if (threadIdx.x == 0) {  // into the slot that the last barrier freed
      fence_proxy_async_smem();
      ring_issue<R>(g, src, ahead, end, p.H, slot == 0 ? g.slots - 1 : slot - 1);
      ahead += step;
    }
    const bool ok = mbar_wait(&full[slot], phase, abort, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteRowWait);
    body(row, static_cast<int>(min(static_cast<long long>(R), end - row)),
         g.mem + static_cast<size_t>(slot) * tensors * g.chunks, g.chunks);
    if (__syncthreads_or(!ok)) break;
    if (++slot == g.slots) {
      slot = 0;
      phase ^= 1;
    }
  }
  if (*abort && threadIdx.x == 0) {  // copies still in flight into this CTA's memory: groups from `row` on
    for (; row < end && row < ahead; row += step) {
      int ignored = 0;
      if (!mbar_wait(&full[slot], phase, &ignored, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteRowDrain)) break;
      if (++slot == g.slots) {
        slot = 0;
        phase ^= 1;
      }
    }
  }
}

// A thread's columns of the vectors: constant over a CTA's rows, as all of them belong to one modulation row.
template <int C>
struct Vecs {
  uint64_t gw[C / 2], mul[C / 2], add[C / 2];  // gate * post_w, mul, add (1, 1 and 0 where absent)
};
template <int C>
VOMNI_DEV void times(const float* p, const bool (&in)[C / 8], int stride, uint64_t (&v)[C / 2]) {
#pragma unroll
  for (int j = 0; j < C / 8; ++j)
    if (in[j]) {
      float t[8];
      load8(p + j * stride, t);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * j + i] = f2_mul(v[4 * j + i], f2_pack(t[2 * i], t[2 * i + 1]));
    }
}
template <int C>
VOMNI_DEV void load_vecs(const Params& p, long long mod, int c, int stride, const bool (&in)[C / 8], Vecs<C>& w) {
  const uint64_t one = both(1.f);
#pragma unroll
  for (int i = 0; i < C / 2; ++i) {
    w.gw[i] = w.mul[i] = one;
    w.add[i] = p.add ? one : 0ull;
  }
  if (p.gate) times<C>(p.gate + mod * p.gate_step + c, in, stride, w.gw);
  if (p.post_w) times<C>(p.post_w + c, in, stride, w.gw);
  if (p.mul) times<C>(p.mul + mod * p.mul_step + c, in, stride, w.mul);
  if (p.add) times<C>(p.add + mod * p.add_step + c, in, stride, w.add);
}

// One group of R rows, forward. load(t, r, v): the thread's values of row r of tensor t (0 x, 1 residual; zero behind the
// row's end); store(t, r, v): to output t.
template <int R, int NV, int kLanes, typename Load, typename Store>
VOMNI_DEV void forward_rows(const Params& p, const Vecs<NV * 8>& w, const bool (&in)[NV], float (*buf)[kBuf], int& turn,
                            Load&& load, Store&& store) {
  constexpr int C = NV * 8;
  Vals<R, C> x;
#pragma unroll
  for (int r = 0; r < R; ++r) load(p.x ? 0 : 1, r, x.v[r]);
  if (p.x) {
    normalise<R, C, kLanes>(x, p.post, in, p, buf, turn);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      uint64_t res[C / 2];
      load(1, r, res);
#pragma unroll
      for (int i = 0; i < C / 2; ++i) x.v[r][i] = f2_fma(x.v[r][i], w.gw[i], res[i]);
      store(0, r, x.v[r]);
    }
  }
  normalise<R, C, kLanes>(x, p.norm, in, p, buf, turn);
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int i = 0; i < C / 2; ++i) x.v[r][i] = f2_fma(x.v[r][i], w.mul[i], w.add[i]);
    store(1, r, x.v[r]);
  }
}

// One group of R rows, backward. load(t, r, v): the thread's values of row r of tensor t (0 x, 1 residual_out, 2 d_res,
// 3 d_out; zero behind the row's end); store(t, r, v): to output t. x and residual_out are read from the
// slot again for each of their statistics instead of being kept: the accumulators and vectors leave registers for two
// tensors of values.
// kPost, kNorm: the kinds, or kAsked to go by the call's; kAll: x, d_res and d_out are all there.
template <int R, int NV, int kLanes, int kPost, int kNorm, bool kAll, typename Load, typename Store>
VOMNI_DEV void backward_rows(const Params& p, const Vecs<NV * 8>& w, const bool (&in)[NV], float (*buf)[kBuf], int& turn,
                             uint64_t (&sum_a)[NV * 4], uint64_t (&sum_m)[NV * 4], uint64_t (&sum_d)[NV * 4], Load&& load,
                             Store&& store) {
  constexpr int C = NV * 8, P = C / 2;
  // statistics of both tensors: 2 r the residual's row r, 2 r + 1 x's
  float mean[2 * R] = {}, rstd[2 * R], s[2 * R];
  const bool has_x = kAll || p.x, has_out = kAll || p.d_out, has_res = kAll || p.d_res;
  const int kind[2] = {kNorm != kAsked ? kNorm : has_out ? p.norm : kNone, kPost != kAsked ? kPost : has_x ? p.post : kNone};
  auto centred = [&](int q, int r, uint64_t (&v)[P]) {
    load(q ? 0 : 1, r, v);
    centre<NV>(v, mean[2 * r + q], in);
  };
  auto hat = [&](int q, int r, uint64_t (&v)[P]) {
    centred(q, r, v);
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = f2_mul(v[i], both(rstd[2 * r + q]));
  };
  if (kind[0] == kLayer || kind[1] == kLayer) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        s[2 * r + q] = 0.f;
        if (kind[q] != kLayer) continue;
        uint64_t v[P];
        load(q ? 0 : 1, r, v);
        uint64_t t = v[0];
#pragma unroll
        for (int i = 1; i < P; ++i) t = f2_add(t, v[i]);
        s[2 * r + q] = halves_sum(t);
      }
    row_sum<2 * R, kLanes>(s, buf, turn);
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) mean[i] = s[i] * p.inv_h;
  }
  if (kind[0] != kNone || kind[1] != kNone) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        s[2 * r + q] = 0.f;
        if (kind[q] == kNone) continue;
        uint64_t v[P];
        centred(q, r, v);
        uint64_t t = f2_mul(v[0], v[0]);
#pragma unroll
        for (int i = 1; i < P; ++i) t = f2_fma(v[i], v[i], t);
        s[2 * r + q] = halves_sum(t);
      }
    row_sum<2 * R, kLanes>(s, buf, turn);
  }
#pragma unroll
  for (int i = 0; i < 2 * R; ++i) rstd[i] = kind[i & 1] == kNone ? 1.f : rsqrtf(s[i] * p.inv_h + p.eps);

  // the sums that normalise's gradient needs of g and g * hat
  auto pair_sums = [&](int r, const uint64_t (&g)[P], const uint64_t (&h)[P]) {
    uint64_t t = g[0], u = f2_mul(g[0], h[0]);
#pragma unroll
    for (int i = 1; i < P; ++i) {
      t = f2_add(t, g[i]);
      u = f2_fma(g[i], h[i], u);
    }
    s[2 * r] = halves_sum(t);
    s[2 * r + 1] = halves_sum(u);
  };
  // g -> rstd (g - [mean g] - hat mean(g hat))
  auto behind = [&](int q, int r, uint64_t (&g)[P], const uint64_t (&h)[P]) {
    const float k = rstd[2 * r + q];
    const uint64_t c1 = both(-k * (s[2 * r + 1] * p.inv_h)), k2 = both(k);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const uint64_t c0 = both(in[j] && kind[q] == kLayer ? -k * (s[2 * r] * p.inv_h) : 0.f);
#pragma unroll
      for (int i = 4 * j; i < 4 * j + 4; ++i) g[i] = f2_fma(g[i], k2, f2_fma(h[i], c1, c0));
    }
  };
  uint64_t d[R][P], h[R][P], v[P];  // h: the normalised rows of the tensor at hand
  if (has_out) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      hat(0, r, h[r]);
      load(3, r, d[r]);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        sum_m[i] = f2_fma(d[r][i], h[r][i], sum_m[i]);
        sum_d[i] = f2_add(sum_d[i], d[r][i]);
        d[r][i] = f2_mul(d[r][i], w.mul[i]);
      }
      pair_sums(r, d[r], h[r]);
    }
    if (kind[0] != kNone) {
      row_sum<2 * R, kLanes>(s, buf, turn);
#pragma unroll
      for (int r = 0; r < R; ++r) behind(0, r, d[r], h[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (!has_out) {
      load(2, r, d[r]);
    } else if (has_res) {
      load(2, r, v);
#pragma unroll
      for (int i = 0; i < P; ++i) d[r][i] = f2_add(d[r][i], v[i]);
    }
    store(1, r, d[r]);
    if (!has_x) continue;
    hat(1, r, h[r]);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      sum_a[i] = f2_fma(d[r][i], h[r][i], sum_a[i]);
      d[r][i] = f2_mul(d[r][i], w.gw[i]);
    }
    pair_sums(r, d[r], h[r]);
  }
  if (!has_x) return;
  if (kind[1] != kNone) row_sum<2 * R, kLanes>(s, buf, turn);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (kind[1] != kNone) behind(1, r, d[r], h[r]);
    store(0, r, d[r]);
  }
}

VOMNI_DEV void unpack_pairs(const uint4& w, uint64_t* v) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = f2_pack(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
}
VOMNI_DEV uint4 pack_pairs(const uint64_t* v) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    f2_unpack(v[i], a, b);
    u[i] = pack_bf16x2(a, b);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

template <int C>
VOMNI_DEV void store_sums(float* part, int pitch, int stride, const bool (&in)[C / 8], const uint64_t (&a)[C / 2],
                          const uint64_t (&m)[C / 2], const uint64_t (&d)[C / 2]) {
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    const uint64_t(&s)[C / 2] = q == 0 ? a : q == 1 ? m : d;
#pragma unroll
    for (int j = 0; j < C / 8; ++j) {
      if (!in[j]) continue;
      ulonglong2* at = reinterpret_cast<ulonglong2*>(part + static_cast<size_t>(q) * pitch + j * stride);
      at[0] = make_ulonglong2(s[4 * j], s[4 * j + 1]);
      at[1] = make_ulonglong2(s[4 * j + 2], s[4 * j + 3]);
    }
  }
}

// A CTA takes R rows at a time; a thread owns chunks (8 columns) threadIdx.x + j * blockDim.x, j < NV.
// kFull: the threads' chunks tile the row exactly, so none carries a predicate.
template <int R, int NV, int kMaxThreads, bool kFull, bool kBackward, int kPost = kAsked, int kNorm = kAsked, bool kAll = false>
__global__ void __launch_bounds__(kMaxThreads, 1) sandwich_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kMaxSlots];
  __shared__ int abort_flag;
  __shared__ __align__(16) float buf[2][kBuf];
  for (int i = threadIdx.x; i < 2 * kBuf; i += blockDim.x) buf[i / kBuf][i % kBuf] = 0.f;  // walk_rows begins with a barrier
  constexpr int C = NV * 8;
  int turn = 0;
  const int c = threadIdx.x * 8, stride = blockDim.x * 8;
  bool in[NV];
  // Of two chunks the first is always there (shape_of: threads <= H / 8 then). Not in the backward pass of one row at a time,
  // which spills without the predicates: 16384 x 8192 430 us instead of 399, forward 223 instead of 238.
#pragma unroll
  for (int j = 0; j < NV; ++j) in[j] = kFull || (NV > 1 && j == 0 && !kBackward) || c + j * stride < p.H;
  const __nv_bfloat16* src[4] = {p.x, (kBackward && !p.d_out) ? nullptr : p.residual, p.d_res, p.d_out};
  int at[4], tensors = 0;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    at[t] = kAll ? t : tensors;
    tensors = kAll ? 4 : tensors + (src[t] != nullptr);
  }
  Vecs<C> w;
  load_vecs<C>(p, blockIdx.y, c, stride, in, w);
  uint64_t sum_a[C / 2] = {}, sum_m[C / 2] = {}, sum_d[C / 2] = {};
  walk_rows<R>(p, src, tensors, smem, full, &abort_flag, [&](long long row, int rows, uint4* slot, int chunks) {
    const int pitch = p.H >> 3;
    if (R > 1 && rows < R) {  // the last group: zeros in place of the missing rows (a thread reads only its own chunks)
      for (int t = 0; t < tensors; ++t)
        for (int r = rows; r < R; ++r)
#pragma unroll
          for (int j = 0; j < NV; ++j)
            if (in[j]) slot[t * chunks + r * pitch + threadIdx.x + j * blockDim.x] = make_uint4(0, 0, 0, 0);
    }
    auto load = [&](int t, int r, uint64_t (&x)[C / 2]) {
      const uint4* s = slot + at[t] * chunks + r * pitch + threadIdx.x;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (in[j]) v = s[j * blockDim.x];
        unpack_pairs(v, &x[4 * j]);
      }
    };
    auto store = [&](int t, int r, const uint64_t (&x)[C / 2]) {
      __nv_bfloat16* out = (t ? p.out1 : p.out0) + (row + r) * p.H + c;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (in[j] && (R == 1 || r < rows)) __stcs(reinterpret_cast<uint4*>(out + j * stride), pack_pairs(&x[4 * j]));
    };
    if constexpr (kBackward)
      backward_rows<R, NV, 0, kPost, kNorm, kAll>(p, w, in, buf, turn, sum_a, sum_m, sum_d, load, store);
    else
      forward_rows<R, NV, 0>(p, w, in, buf, turn, load, store);
  });
  if constexpr (kBackward) {
    pdl_trigger();  // the sums' launch may get ready while the last rows end
    store_sums<C>(p.parts + (static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x) * 3 * p.H + c, p.H, stride, in, sum_a,
                  sum_m, sum_d);
  }
}

// ---------------------------------------------------------------- long calls' backward pass
// The backward pass of calls with a branch and both gradients over many rows: R rows at a time, like backward_rows, but the
// statistics of the next R rows are summed along with this group's gradients, so that a group costs two barriers (the
// second also frees its slots) instead of five. For that x and residual_out of the next group are there a group early: they have
// three slots, the gradients two. One CTA of 10 warps an SM has nothing else to
// issue around a barrier: 32760 x 5120 356 us instead of 383 with sandwich_kernel, 0.86 of the measured copy rate. Several CTAs an SM
// hide that by themselves (32760 x 1536: 125 us with either). One row at a time, where each row takes the two
// barriers, it is slower (16384 x 8192: 481 us instead of 397).
template <int R, int NV, int kMaxThreads, bool kFull, int kPost, int kNorm>
__global__ void __launch_bounds__(kMaxThreads, 1) sandwich_bwd_kernel(const __grid_constant__ Params p) {
  constexpr int C = NV * 8, P = C / 2;
  constexpr bool kMeans = kPost == kLayer || kNorm == kLayer, kSquares = kPost != kNone || kNorm != kNone;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[5];  // rows' slots, gradients' slots
  __shared__ int abort_flag;
  __shared__ __align__(16) float buf[2][kBuf];
  for (int i = threadIdx.x; i < 2 * kBuf; i += blockDim.x) buf[i / kBuf][i % kBuf] = 0.f;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 5; ++i) mbar_init(&full[i], 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  const int c = threadIdx.x * 8, stride = blockDim.x * 8, pitch = p.H >> 3, chunks = R * pitch;
  const long long begin = static_cast<long long>(blockIdx.y) * p.rows_per_mod, end = begin + p.rows_per_mod;
  const long long first = begin + static_cast<long long>(blockIdx.x) * R, step = static_cast<long long>(gridDim.x) * R;
  uint4* const mem = reinterpret_cast<uint4*>(smem);  // [3][x, residual_out][chunks], [2][d_res, d_out][chunks]
  auto rows_slot = [&](int s) { return mem + s * 2 * chunks; };
  auto grads_slot = [&](int s) { return mem + (6 + s * 2) * chunks; };
  auto issue = [&](const __nv_bfloat16* a, const __nv_bfloat16* b, long long row, uint4* dst, uint64_t* bar) {
    if (row >= end) return;
    const uint32_t bytes = static_cast<uint32_t>(min(static_cast<long long>(R), end - row)) * p.H * 2u;
    mbar_expect_tx(bar, 2 * bytes);
    bulk_g2s(dst, a + row * p.H, bytes, bar);
    bulk_g2s(dst + chunks, b + row * p.H, bytes, bar);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < 3; ++s) {
      issue(p.x, p.residual, first + s * step, rows_slot(s), &full[s]);
      if (s < 2) issue(p.d_res, p.d_out, first + s * step, grads_slot(s), &full[3 + s]);
    }
  }
  bool in[NV];
  // of two chunks the first is always there (shape_of: threads <= H / 8 then): 16384 x 5000 195 us instead of 227
#pragma unroll
  for (int j = 0; j < NV; ++j) in[j] = kFull || (NV > 1 && j == 0) || c + j * stride < p.H;
  Vecs<C> w;
  load_vecs<C>(p, blockIdx.y, c, stride, in, w);
  uint64_t sum_a[P] = {}, sum_m[P] = {}, sum_d[P] = {};
  int turn = 0;
  bool ok = true;
  auto wait = [&](int bar, uint32_t use) {
    ok = mbar_wait(&full[bar], use & 1, &abort_flag, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteRowWait) && ok;
  };
  auto clear_missing = [&](uint4* slot, long long row) {  // zeros in place of rows behind the last (a thread reads only its chunks)
    if (R == 1 || end - row >= R) return;
    for (int t = 0; t < 2; ++t)
      for (int r = static_cast<int>(end - row); r < R; ++r)
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (in[j]) slot[t * chunks + r * pitch + threadIdx.x + j * blockDim.x] = make_uint4(0, 0, 0, 0);
  };
  auto load = [&](const uint4* slot, int t, int r, uint64_t (&v)[P]) {
    const uint4* s = slot + t * chunks + r * pitch + threadIdx.x;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (in[j]) u = s[j * blockDim.x];
      unpack_pairs(u, &v[4 * j]);
    }
  };
  // Partial sums of a group's statistics; of row r: 2 r residual_out's, 2 r + 1 x's.
  constexpr int kKind[2] = {kNorm, kPost};
  auto sums_of = [&](const uint4* slot, float* s) {
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) {
      s[i] = 0.f;
      if (kKind[i & 1] != kLayer) continue;
      uint64_t v[P];
      load(slot, i & 1 ? 0 : 1, i >> 1, v);
      uint64_t t = v[0];
#pragma unroll
      for (int k = 1; k < P; ++k) t = f2_add(t, v[k]);
      s[i] = halves_sum(t);
    }
  };
  auto squares_of = [&](const uint4* slot, const float (&mean)[2 * R], float* s) {
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) {
      s[i] = 0.f;
      if (kKind[i & 1] == kNone) continue;
      uint64_t v[P];
      load(slot, i & 1 ? 0 : 1, i >> 1, v);
      if (kKind[i & 1] == kLayer) centre<NV>(v, mean[i], in);
      uint64_t t = f2_mul(v[0], v[0]);
#pragma unroll
      for (int k = 1; k < P; ++k) t = f2_fma(v[k], v[k], t);
      s[i] = halves_sum(t);
    }
  };
  float mean[2 * R] = {}, rstd[2 * R], next_mean[2 * R] = {};
  auto deviations = [&](const float* s) {
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) rstd[i] = kKind[i & 1] == kNone ? 1.f : rsqrtf(s[i] * p.inv_h + p.eps);
  };
  auto hat = [&](const uint4* slot, int i, uint64_t (&v)[P]) {  // normalised row i >> 1 of residual_out or x
    load(slot, i & 1 ? 0 : 1, i >> 1, v);
    if (kKind[i & 1] == kLayer) centre<NV>(v, mean[i], in);
    if (kKind[i & 1] != kNone) {
#pragma unroll
      for (int k = 0; k < P; ++k) v[k] = f2_mul(v[k], both(rstd[i]));
    }
  };
  auto pair_sums = [&](const uint64_t (&g)[P], const uint64_t (&h)[P], float* s) {
    uint64_t t = g[0], u = f2_mul(g[0], h[0]);
#pragma unroll
    for (int k = 1; k < P; ++k) {
      t = f2_add(t, g[k]);
      u = f2_fma(g[k], h[k], u);
    }
    s[0] = halves_sum(t);
    s[1] = halves_sum(u);
  };
  auto behind = [&](int i, uint64_t (&g)[P], const uint64_t (&h)[P], const float* s) {
    const float k = rstd[i];
    const uint64_t c1 = both(-k * (s[1] * p.inv_h)), k2 = both(k);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const uint64_t c0 = both(in[j] && kKind[i & 1] == kLayer ? -k * (s[0] * p.inv_h) : 0.f);
#pragma unroll
      for (int q = 4 * j; q < 4 * j + 4; ++q) g[q] = f2_fma(g[q], k2, f2_fma(h[q], c1, c0));
    }
  };
  {  // the first group's statistics
    wait(0, 0);
    clear_missing(rows_slot(0), first);
    float s[2 * R];
    if (kMeans) {
      sums_of(rows_slot(0), s);
      row_sum<2 * R, 0>(s, buf, turn);
#pragma unroll
      for (int i = 0; i < 2 * R; ++i) mean[i] = s[i] * p.inv_h;
    }
    if (kSquares) {
      squares_of(rows_slot(0), mean, s);
      row_sum<2 * R, 0>(s, buf, turn);
    }
    deviations(s);
  }
  long long row = first;
  int slot = 0, next = 1, gslot = 0;  // slots of this group's rows, the next one's and this group's gradients
  uint32_t use = 0, next_use = 0, guse = 0;
  for (; row < end; row += step) {
    const bool more = row + step < end;
    const uint4 *xr = rows_slot(slot), *xn = rows_slot(next), *g = grads_slot(gslot);
    wait(3 + gslot, guse);
    clear_missing(grads_slot(gslot), row);
    if (more) {
      wait(next, next_use);
      clear_missing(rows_slot(next), row + step);
    }
    auto store = [&](__nv_bfloat16* out, int r, const uint64_t (&v)[P]) {
      out += (row + r) * p.H + c;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (in[j] && (R == 1 || row + r < end)) __stcs(reinterpret_cast<uint4*>(out + j * stride), pack_pairs(&v[4 * j]));
    };
    uint64_t d[R][P], h[R][P], v[P];
    float s[4 * R] = {};  // this group's sums, the next one's
#pragma unroll
    for (int r = 0; r < R; ++r) {
      hat(xr, 2 * r, h[r]);
      load(g, 1, r, d[r]);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        sum_m[i] = f2_fma(d[r][i], h[r][i], sum_m[i]);
        sum_d[i] = f2_add(sum_d[i], d[r][i]);
        d[r][i] = f2_mul(d[r][i], w.mul[i]);
      }
      if (kNorm != kNone) pair_sums(d[r], h[r], &s[2 * r]);
    }
    if constexpr (kMeans) {
      if (more) sums_of(xn, s + 2 * R);
      row_sum<4 * R, 0>(s, buf, turn);
#pragma unroll
      for (int i = 0; i < 2 * R; ++i) next_mean[i] = s[2 * R + i] * p.inv_h;
    } else if constexpr (kNorm != kNone) {
      float t[2 * R];
#pragma unroll
      for (int i = 0; i < 2 * R; ++i) t[i] = s[i];
      row_sum<2 * R, 0>(t, buf, turn);
#pragma unroll
      for (int i = 0; i < 2 * R; ++i) s[i] = t[i];
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (kNorm != kNone) behind(2 * r, d[r], h[r], &s[2 * r]);
      load(g, 0, r, v);
#pragma unroll
      for (int i = 0; i < P; ++i) d[r][i] = f2_add(d[r][i], v[i]);
      store(p.out1, r, d[r]);
      hat(xr, 2 * r + 1, h[r]);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        sum_a[i] = f2_fma(d[r][i], h[r][i], sum_a[i]);
        d[r][i] = f2_mul(d[r][i], w.gw[i]);
      }
      s[2 * r] = s[2 * r + 1] = 0.f;
      if (kPost != kNone) pair_sums(d[r], h[r], &s[2 * r]);
    }
    bool bad;
    if constexpr (kSquares) {
      if (more) squares_of(xn, next_mean, s + 2 * R);
      bad = row_sum<4 * R, 0, true>(s, buf, turn, !ok);
    } else {
      bad = __syncthreads_or(!ok);
    }
    if (bad) break;
    if (threadIdx.x == 0) {  // every thread has read this group's slots
      fence_proxy_async_smem();
      issue(p.d_res, p.d_out, row + 2 * step, grads_slot(gslot), &full[3 + gslot]);
      issue(p.x, p.residual, row + 3 * step, rows_slot(slot), &full[slot]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (kPost != kNone) behind(2 * r + 1, d[r], h[r], &s[2 * r]);
      store(p.out0, r, d[r]);
    }
#pragma unroll
    for (int i = 0; i < 2 * R; ++i) mean[i] = next_mean[i];
    deviations(s + 2 * R);
    slot = next;
    use = next_use;
    if (++next == 3) {
      next = 0;
      ++next_use;
    }
    if (++gslot == 2) {
      gslot = 0;
      ++guse;
    }
  }
  if (abort_flag && threadIdx.x == 0) {  // copies still in flight into this CTA's memory: of groups from `row` on
    int ignored = 0;
    for (int i = 0; i < 3 && row + i * step < end; ++i) {
      mbar_wait(&full[slot], use & 1, &ignored, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteRowDrain);
      if (i < 2) mbar_wait(&full[3 + gslot], guse & 1, &ignored, p.status, VOMNI_DEV_TIMEOUT_BASE + kSiteRowDrain);
      if (++slot == 3) {
        slot = 0;
        ++use;
      }
      if (++gslot == 2) {
        gslot = 0;
        ++guse;
      }
    }
  }
  pdl_trigger();  // the sums' launch may get ready while the last rows end
  store_sums<C>(p.parts + (static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x) * 3 * p.H + c, p.H, stride, in, sum_a,
                sum_m, sum_d);
}

// Short rows (H <= 256): kLanes lanes a row, 32 / kLanes rows a warp, straight from global memory, the next rows' loads
// under way meanwhile. The column sums are added in the CTA, in order: a part per warp left the sums' kernel thousands to add.
// Backward (with 6 us of two launches): 200000 x 128 68 us instead of 172 with a row and a part a warp and no loads ahead, 98280 x 256
// 68 instead of 102, 20000 x 64 14 instead of 41.
constexpr int kRowWarps = 8;
template <bool kBackward, int kLanes>
__global__ void __launch_bounds__(32 * kRowWarps) sandwich_warp_kernel(const __grid_constant__ Params p) {
  constexpr int kRows = 32 / kLanes;  // of a warp
  const int sub = threadIdx.x / kLanes, c = threadIdx.x % kLanes * 8;
  const bool in[1] = {c < p.H};
  const long long end = (static_cast<long long>(blockIdx.y) + 1) * p.rows_per_mod;
  Vecs<8> w;
  load_vecs<8>(p, blockIdx.y, c, 0, in, w);
  uint64_t sum_a[4] = {}, sum_m[4] = {}, sum_d[4] = {};
  int turn = 0;
  const __nv_bfloat16* src[4] = {p.x, (kBackward && !p.d_out) ? nullptr : p.residual, p.d_res, p.d_out};
  constexpr int kTensors = kBackward ? 4 : 2;
  uint4 next[kTensors];
  auto fetch = [&](long long row) {  // zeros for rows behind the last
#pragma unroll
    for (int t = 0; t < kTensors; ++t) {
      next[t] = make_uint4(0, 0, 0, 0);
      if (in[0] && row < end && src[t]) next[t] = __ldcs(reinterpret_cast<const uint4*>(src[t] + row * p.H + c));
    }
  };
  const int step = static_cast<int>(gridDim.x) * kRowWarps * kRows;
  long long first = static_cast<long long>(blockIdx.y) * p.rows_per_mod + (blockIdx.x * kRowWarps + threadIdx.y) * kRows;  // the warp's
  fetch(first + sub);
  for (; first < end; first += step) {
    const long long row = first + sub;
    uint4 raw[kTensors];
#pragma unroll
    for (int t = 0; t < kTensors; ++t) raw[t] = next[t];
    fetch(row + step);
    auto load = [&](int t, int, uint64_t (&x)[4]) { unpack_pairs(raw[t], x); };
    auto store = [&](int t, int, const uint64_t (&x)[4]) {
      if (in[0] && row < end) __stcs(reinterpret_cast<uint4*>((t ? p.out1 : p.out0) + row * p.H + c), pack_pairs(x));
    };
    if constexpr (kBackward)
      backward_rows<1, 1, kLanes, kAsked, kAsked, false>(p, w, in, nullptr, turn, sum_a, sum_m, sum_d, load, store);
    else
      forward_rows<1, 1, kLanes>(p, w, in, nullptr, turn, load, store);
  }
  if constexpr (kBackward) {
    pdl_trigger();
    __shared__ __align__(16) float red[kRowWarps * kRows][3][8 * kLanes];
    const bool every[1] = {true};
    store_sums<8>(&red[threadIdx.y * kRows + sub][0][0] + c, 8 * kLanes, 0, every, sum_a, sum_m, sum_d);
    __syncthreads();
    float* part = p.parts + (static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x) * 3 * p.H;
    for (int i = threadIdx.y * 32 + threadIdx.x; i < 3 * p.H; i += 32 * kRowWarps) {
      const int q = i / p.H, col = i - q * p.H;
      float t = red[0][q][col];
#pragma unroll
      for (int k = 1; k < kRowWarps * kRows; ++k) t += red[k][q][col];
      part[i] = t;
    }
  }
}

struct SumParams {
  float* parts;  // [n_mod][lanes][3][H]
  const float* gate;
  const float* post_w;
  long long gate_step;
  int H, lanes, n_mod, per;  // per: kPer* flags
  int mods;                  // modulation rows of a range
  float *dgate, *dpost_w, *dmul, *dadd;
};

// What the sum over all modulation rows gives: the shared vectors' gradients. For A it was weighed with a gate per
// modulation row; a shared gate is constant in it.
VOMNI_DEV void store_shared(const SumParams& p, int q, int col, float sum) {
  float* out = q == 0 ? p.dgate : q == 1 ? p.dmul : p.dadd;
  if (q == 0) {
    const bool per = p.per & kPerGate;
    if (p.dpost_w) p.dpost_w[col] = per || !p.gate ? sum : sum * p.gate[col];
    if (out && !per) out[col] = p.post_w ? sum * p.post_w[col] : sum;
  } else if (out && !(p.per & (q == 1 ? kPerMul : kPerAdd))) {
    out[col] = sum;
  }
}

// The gradient of one modulation row, where its vector has one per row; returns what is added over the rows.
VOMNI_DEV float store_row(const SumParams& p, int q, int mod, int col, float t) {
  float* out = q == 0 ? p.dgate : q == 1 ? p.dmul : p.dadd;
  const bool per = p.per & (q == 0 ? kPerGate : q == 1 ? kPerMul : kPerAdd);
  if (per && out) out[static_cast<long long>(mod) * p.H + col] = q == 0 && p.post_w ? t * p.post_w[col] : t;
  return q == 0 && per && p.gate ? t * p.gate[mod * p.gate_step + col] : t;
}
VOMNI_DEV bool asked(const SumParams& p, int q) { return q == 0 ? p.dgate || p.dpost_w : q == 1 ? p.dmul != nullptr : p.dadd != nullptr; }

// 32 columns x 32 lanes a CTA; blockIdx.y: A, M or D. Sums each modulation row's parts in the order lane, lane + 32, ...,
// then the 32 lanes as a tree, and forms the outputs; those shared by the modulation rows are added over them in order.
// (With 8 lanes it took 13 us for 334 parts of 1536 columns, more than the kernel before it.)
__global__ void __launch_bounds__(1024) sandwich_sum_kernel(const __grid_constant__ SumParams p) {
  __shared__ float red[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x, q = blockIdx.y;
  const bool in = col < p.H;
  pdl_wait();  // launched as a dependent of the rows' kernel
  if (!asked(p, q)) return;
  float sum = 0.f;
  const int mine = blockIdx.x * 32 + threadIdx.y;  // the column whose lanes this warp adds
  for (int mod = 0; mod < p.n_mod; ++mod) {
    float s = 0.f;
    if (in) {
      const float* at = p.parts + (static_cast<long long>(mod) * p.lanes * 3 + q) * p.H + col;
#pragma unroll 4
      for (int l = threadIdx.y; l < p.lanes; l += 32) s += at[static_cast<long long>(l) * 3 * p.H];
    }
    red[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    float t = red[threadIdx.x][threadIdx.y];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (threadIdx.x == 0 && mine < p.H) sum += store_row(p, q, mod, mine, t);
    __syncthreads();
  }
  if (threadIdx.x == 0 && mine < p.H) store_shared(p, q, mine, sum);
}

// The same for many modulation rows, of which each then has few parts: a thread per column and range of `mods` rows
// (blockIdx.z). Its sum over the rows goes to the range's first part (read by no other thread), sandwich_shared_kernel adds the ranges'.
__global__ void __launch_bounds__(256) sandwich_ranges_kernel(const __grid_constant__ SumParams p) {
  const int col = blockIdx.x * blockDim.x + threadIdx.x, q = blockIdx.y;
  pdl_wait();  // launched as a dependent of the rows' kernel
  if (col >= p.H || !asked(p, q)) return;
  const int first = blockIdx.z * p.mods, last = min(first + p.mods, p.n_mod);
  float sum = 0.f;
  for (int mod = first; mod < last; ++mod) {
    const float* at = p.parts + (static_cast<long long>(mod) * p.lanes * 3 + q) * p.H + col;
    float t = 0.f;
#pragma unroll 8
    for (int l = 0; l < p.lanes; ++l) t += at[static_cast<long long>(l) * 3 * p.H];
    sum += store_row(p, q, mod, col, t);
  }
  p.parts[(static_cast<long long>(first) * p.lanes * 3 + q) * p.H + col] = sum;
}
__global__ void __launch_bounds__(256) sandwich_shared_kernel(const __grid_constant__ SumParams p) {
  const int col = blockIdx.x * blockDim.x + threadIdx.x, q = blockIdx.y;
  if (col >= p.H || !asked(p, q)) return;
  float sum = 0.f;
  for (int mod = 0; mod < p.n_mod; mod += p.mods) sum += p.parts[(static_cast<long long>(mod) * p.lanes * 3 + q) * p.H + col];
  store_shared(p, q, col, sum);
}

// How a call is laid out: a row or more per warp, or R rows at a time per CTA with NV chunks a thread.
struct Shape {
  int row_lanes;  // of a row that is part of a warp, else 0
  int nv, rows, threads;  // rows: R
  int lanes;              // CTAs that share a modulation row's tokens
  unsigned blocks;        // gridDim.x
  int slots;
  size_t smem;
};
Shape shape_of(long long rows_per_mod, long long n_mod, int h, int tensors, bool backward) {
  Shape s = {};
  const int chunks = h / 8;
  s.row_lanes = chunks <= 8 ? 8 : chunks <= 16 ? 16 : chunks <= 32 ? 32 : 0;
  if (s.row_lanes) {
    const int rows = kRowWarps * 32 / s.row_lanes;  // of a CTA at a time; two or four CTAs fit an SM
    const long long need = (rows_per_mod + rows - 1) / rows;
    const long long cap = std::max(1ll, num_sms() * (backward ? 2ll : 4ll) / n_mod);
    s.blocks = static_cast<unsigned>(need < cap ? need : cap);
    s.lanes = static_cast<int>(s.blocks);
    return s;
  }
  // Few rows: one at a time, so that they spread over the device. Else a thread of the backward pass takes two chunks
  // of a row and two rows, of the forward pass one and four (kernel_of says why).
  const bool many = rows_per_mod * n_mod >= 4ll * num_sms();
  s.nv = chunks > 640 || (backward && many) ? 2 : 1;
  s.threads = ((chunks + s.nv - 1) / s.nv + 31) / 32 * 32;
  s.rows = chunks > 640 || !many ? 1 : backward ? 2 : 4;
  const size_t slot = static_cast<size_t>(s.rows) * h * 2 * tensors;
  // What the registers hold: 640 threads an SM forward, 320 backward. The quotient is rounded down, so just over half of them one CTA
  // is left with an SM to itself (backward, 16384 rows: 3000 columns 1.7 times the bytes' time, 5120 1.2 times); rows over 5120 columns go one
  // at a time (8192 columns 1.6 times).
  const int per_sm = std::max(1, std::min((backward && many ? 320 : 640) / s.threads, 8));
  const size_t room = (kSmemPerSm / per_sm);
  s.slots = static_cast<int>(std::max<size_t>(2, std::min<size_t>(kMaxSlots, room / slot)));
  s.smem = slot * s.slots;
  const long long need = (rows_per_mod + s.rows - 1) / s.rows;
  // Rounded down: one CTA more than fits would run after all the others (3 x 1000 x 5120 backward: 96 us with 150 CTAs, 70 with 147).
  // Between half of what fits and all of it each modulation row gets one CTA and the rest idles, and past all of it the last ones do run
  // after the others: backward, 200 tokens of 5120 columns each, 74 rows 163 us, 75 to 148 rows 305, 149 to 296 rows 600.
  const long long cap = std::max(1ll, static_cast<long long>(num_sms()) * per_sm / n_mod);
  s.blocks = static_cast<unsigned>(need < cap ? need : cap);
  s.lanes = static_cast<int>(s.blocks);
  return s;
}

typedef void (*Kernel)(Params);

bool all_given(const Params& p) { return p.x && p.d_res && p.d_out; }

// The backward kernels that know their norms at compile time (430 us instead of 574 at 32760 x 5120 when both were the same
// kernel): those of a call with a branch and both gradients. Two rows at a time: sandwich_bwd_kernel; one: sandwich_kernel.
template <int R, bool kFull, int kPost, int kNorm>
Kernel backward_kind() {
  if constexpr (R == 2)
    return sandwich_bwd_kernel<2, 2, 320, kFull, kPost, kNorm>;
  else
    return sandwich_kernel<1, 2, 512, kFull, true, kPost, kNorm, true>;
}
template <int R, bool kFull>
Kernel backward_of(const Params& p) {
  switch (p.post * 3 + p.norm) {
    case 0: return backward_kind<R, kFull, 0, 0>();
    case 1: return backward_kind<R, kFull, 0, 1>();
    case 2: return backward_kind<R, kFull, 0, 2>();
    case 3: return backward_kind<R, kFull, 1, 0>();
    case 4: return backward_kind<R, kFull, 1, 1>();
    case 5: return backward_kind<R, kFull, 1, 2>();
    case 6: return backward_kind<R, kFull, 2, 0>();
    case 7: return backward_kind<R, kFull, 2, 1>();
    default: return backward_kind<R, kFull, 2, 2>();
  }
}

// Rows at a time and chunks a thread. The reductions cost a warp the same for one value a thread as for many and all
// warps wait for each other in them, so more of both is better while registers and shared memory last. Measured at
// 32760 x 5120: forward 393 / 299 / 228 us with 1 / 2 / 4 rows of one chunk; backward (sandwich_kernel) 402 us with two rows
// of one chunk (640 threads), 383 us with two rows of two (320), 624 us with one row of two, 740 us with one row of four.
template <bool kBackward>
Kernel kernel_of(const Params& p, const Shape& s) {
  const bool full = s.threads * s.nv * 8 == p.H;
  if constexpr (kBackward) {
    const bool all = all_given(p);
    if (s.rows == 2) return !all ? sandwich_kernel<2, 2, 320, false, true> : full ? backward_of<2, true>(p) : backward_of<2, false>(p);
    if (s.nv == 2) return all ? backward_of<1, false>(p) : sandwich_kernel<1, 2, 512, false, true>;
    return sandwich_kernel<1, 1, 640, false, true>;
  } else {
    if (s.rows == 4) return full ? sandwich_kernel<4, 1, 640, true, false> : sandwich_kernel<4, 1, 640, false, false>;
    if (s.nv == 2) return sandwich_kernel<1, 2, 512, false, false>;
    return sandwich_kernel<1, 1, 640, false, false>;
  }
}

template <bool kBackward>
int launch(Params p, long long n_mod, const Shape& s, cudaStream_t st) {
  p.slots = s.slots;
  p.status = device_status_ptr();
  const dim3 grid(s.blocks, static_cast<unsigned>(n_mod));
  if (s.row_lanes) {
    const Kernel kern = s.row_lanes == 8    ? sandwich_warp_kernel<kBackward, 8>
                        : s.row_lanes == 16 ? sandwich_warp_kernel<kBackward, 16>
                                            : sandwich_warp_kernel<kBackward, 32>;
    kern<<<grid, dim3(32, kRowWarps), 0, st>>>(p);
  } else {
    // sandwich_bwd_kernel: three slots of two tensors and two of the others (at most 200 KB an SM for the CTAs that
    // shape_of counts: per_sm <= 5120 / H)
    const size_t smem = kBackward && s.rows == 2 && all_given(p) ? static_cast<size_t>(10) * s.rows * p.H * 2 : s.smem;
    const Kernel kern = kernel_of<kBackward>(p, s);
    int rc = ensure_max_smem(kern, static_cast<int>(smem));
    if (rc) return rc;
    kern<<<grid, s.threads, smem, st>>>(p);
  }
  VOMNI_CUDA_TRY(cudaGetLastError());
  return VOMNI_OK;
}

int check(long long rows, int h, long long rows_per_mod, int post, int norm, float eps) {
  if (rows <= 0 || rows > 0x7fffffffLL || h <= 0 || h > kMaxH || h % 8) return VOMNI_EBADSHAPE;
  if (rows_per_mod <= 0 || rows % rows_per_mod || rows / rows_per_mod > 65535) return VOMNI_EBADSHAPE;
  if (post < 0 || post > 2 || norm < 0 || norm > 2) return VOMNI_EINVAL;
  if (!(eps > 0.f && eps <= 3.0e38f)) return VOMNI_EINVAL;  // rows behind the last one are zero: eps keeps them finite
  return VOMNI_OK;
}
bool misaligned(const void* a, const void* b = nullptr, const void* c = nullptr, const void* d = nullptr) {
  return (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) |
          reinterpret_cast<uintptr_t>(d)) & 15;
}
void fill(Params& p, const void* x, const void* residual, const float* gate, const float* post_w, const float* mul,
          const float* add, int h, long long rows_per_mod, int per, float eps, int post, int norm) {
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.residual = static_cast<const __nv_bfloat16*>(residual);
  p.gate = gate;
  p.post_w = post_w;
  p.mul = mul;
  p.add = add;
  p.rows_per_mod = rows_per_mod;
  p.gate_step = per & kPerGate ? h : 0;
  p.mul_step = per & kPerMul ? h : 0;
  p.add_step = per & kPerAdd ? h : 0;
  p.H = h;
  p.post = post;
  p.norm = norm;
  p.eps = eps;
  p.inv_h = 1.f / static_cast<float>(h);
}

}  // namespace sandwich
}  // namespace vomni

using namespace vomni;

extern "C" int vomni_sandwich_norm(const void* x, const void* residual, const float* gate, const float* post_weight,
                                   const float* mul, const float* add, long long rows, int h, long long rows_per_mod,
                                   int per_mod, float eps, int post_norm, int norm_type, void* residual_out, void* out,
                                   vomni_stream_t stream) {
  using namespace sandwich;
  if (!residual || !out || (x && !residual_out) || (per_mod & ~7)) return VOMNI_EINVAL;
  if (!x && (gate || post_weight || residual_out)) return VOMNI_EINVAL;
  int rc = check(rows, h, rows_per_mod, post_norm, norm_type, eps);
  if (rc) return rc;
  if (misaligned(x, residual, residual_out, out) || misaligned(gate, post_weight, mul, add)) return VOMNI_EALIGN;
  rc = require_sm100();
  if (rc) return rc;
  Params p = {};
  fill(p, x, residual, gate, post_weight, mul, add, h, rows_per_mod, per_mod, eps, post_norm, norm_type);
  p.out0 = static_cast<__nv_bfloat16*>(residual_out);
  p.out1 = static_cast<__nv_bfloat16*>(out);
  const long long n_mod = rows / rows_per_mod;
  return launch<false>(p, n_mod, shape_of(rows_per_mod, n_mod, h, x ? 2 : 1, false),
                       reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t vomni_sandwich_norm_workspace_bytes(long long rows, int h, long long rows_per_mod) {
  using namespace sandwich;
  if (check(rows, h, rows_per_mod, 0, 0, 1.f)) return 0;
  const long long n_mod = rows / rows_per_mod;
  return static_cast<size_t>(n_mod) * shape_of(rows_per_mod, n_mod, h, 4, true).lanes * 3 * h * sizeof(float);
}

extern "C" int vomni_sandwich_norm_bwd(const void* grad_residual_out, const void* grad_out, const void* x,
                                       const void* residual_out, const float* gate, const float* post_weight,
                                       const float* mul, long long rows, int h, long long rows_per_mod, int per_mod,
                                       float eps, int post_norm, int norm_type, void* dx, void* dresidual, float* dgate,
                                       float* dpost_weight, float* dmul, float* dadd, void* workspace,
                                       size_t workspace_bytes, vomni_stream_t stream) {
  using namespace sandwich;
  if ((!grad_residual_out && !grad_out) || !dresidual || !workspace || (per_mod & ~7)) return VOMNI_EINVAL;
  if (grad_out && !residual_out) return VOMNI_EINVAL;
  if (x ? !dx : (gate || post_weight || dgate || dpost_weight || dx)) return VOMNI_EINVAL;
  int rc = check(rows, h, rows_per_mod, post_norm, norm_type, eps);
  if (rc) return rc;
  const long long n_mod = rows / rows_per_mod;
  if (workspace_bytes < vomni_sandwich_norm_workspace_bytes(rows, h, rows_per_mod)) return VOMNI_EWORKSPACE;
  if (misaligned(x, residual_out, grad_residual_out, grad_out) || misaligned(gate, post_weight, mul, workspace) ||
      misaligned(dx, dresidual))
    return VOMNI_EALIGN;
  rc = require_sm100();
  if (rc) return rc;
  Params p = {};
  fill(p, x, residual_out, gate, post_weight, mul, nullptr, h, rows_per_mod, per_mod, eps, post_norm, norm_type);
  p.d_res = static_cast<const __nv_bfloat16*>(grad_residual_out);
  p.d_out = static_cast<const __nv_bfloat16*>(grad_out);
  p.out0 = static_cast<__nv_bfloat16*>(dx);
  p.out1 = static_cast<__nv_bfloat16*>(dresidual);
  p.parts = static_cast<float*>(workspace);
  const Shape sh = shape_of(rows_per_mod, n_mod, h, 4, true);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  rc = launch<true>(p, n_mod, sh, st);
  if (rc) return rc;
  if (!dgate && !dpost_weight && !dmul && !dadd) return VOMNI_OK;
  SumParams s = {};
  s.parts = p.parts;
  s.gate = gate;
  s.post_w = post_weight;
  s.gate_step = p.gate_step;
  s.H = h;
  s.lanes = sh.lanes;
  s.n_mod = static_cast<int>(n_mod);
  s.per = per_mod;
  s.dgate = dgate;
  s.dpost_w = dpost_weight;
  s.dmul = dmul;
  s.dadd = dadd;
  // sandwich_sum_kernel takes its modulation rows one after another, the other kernel a row's parts; the other one's second launch is
  // 3 us. Whole passes, sum / ranges: 64 x 100 x 1536 (12 parts) 127 / 57 us, 20000 x 1 x 5120 (1) 77 900 / 2200, 4 x 1000 x 5120 (37)
  // 84 / 72, 8 x 333 x 1536 (92) 39 / 37, 4 x 2000 x 128 (74) 18 / 22, 4 x 333 x 1536 (167) 25 / 33.
  const bool many = n_mod >= 4 && s.lanes <= 64;
  s.mods = static_cast<int>((n_mod + 63) / 64);
  const unsigned ranges = static_cast<unsigned>((n_mod + s.mods - 1) / s.mods);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = many ? dim3((h + 255) / 256, 3, ranges) : dim3((h + 31) / 32, 3);
  cfg.blockDim = many ? dim3(256) : dim3(32, 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VOMNI_CUDA_TRY(cudaLaunchKernelEx(&cfg, many ? sandwich_ranges_kernel : sandwich_sum_kernel, s));
  const bool shared = dpost_weight || (dgate && !(per_mod & kPerGate)) || (dmul && !(per_mod & kPerMul)) || (dadd && !(per_mod & kPerAdd));
  if (many && shared) {
    sandwich_shared_kernel<<<dim3((h + 255) / 256, 3), 256, 0, st>>>(s);
    VOMNI_CUDA_TRY(cudaGetLastError());
  }
  return VOMNI_OK;
}
