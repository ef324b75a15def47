// Attention forward for training, of any inputs whose products fp32 holds: the const-max pass, and the rows that its bound does not fit once more
// under their own maximum.
//
// The const-max pass (cm_attn.cu) sums l_i = sum_j exp(s_ij - c_i) under c_i = scale |q_i| max |k_j|. An exponential below 2^-126 is
// flushed to 0, so what a row loses is at most n 2^-126 of l_i: the row is right where l_i >= n 2^-102 (it loses 2^-24 at most), which
// normal q and k of deviation 2 still are. With large norms the largest score lies too far below c_i (normal vectors of
// deviation 3 are: half the rows lose all their probabilities), or, as c_i is held in bf16, so far above it that l_i nears the end
// of fp32. Those rows are found from lse_i - c_i = log l_i and computed again here with a running maximum; all others keep what
// the const-max pass wrote, to the bit.
//
// A CTA of four warps takes 64 rows, 16 a warp, and walks the keys in tiles of 64 through two slots of shared memory: S = Q K^T
// and O += P V with mma.sync, whose fragments of S are those of P, so that P never leaves registers. No barrier waits, no TMEM: this
// pass is for the rows that are left over (230 to 290 TFLOP/s where all are: 32760 tokens of 8 heads 19 ms, 4096 of 40 heads 1.6 ms, of
// deviation 4). P is rounded to bf16 for the product and O divided by the sum of the rounded values,
// as in the const-max pass; lse is the log of the unrounded sum.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "host_util.h"

namespace vomni {
namespace afwd {

constexpr int kD = 128;
constexpr int kRows = 64;   // of a CTA: 16 a warp
constexpr int kKeys = 64;   // of a step
constexpr int kWarps = 4;
constexpr uint32_t kTileBytes = kKeys * kD * 2;  // 16 KB
constexpr uint32_t kSmemBytes = 4 * kTileBytes;  // [2 slots][K, V]
constexpr int kCtasPerSm = 3;

struct Params {
  const __nv_bfloat16 *q, *k, *v;
  long long q_stride, kv_stride;  // of a token, elements
  int s_q, s_kv, h;
  float scale;
  const float* qn2;    // [b * h, s_q]
  const float* kmax2;  // [b * h]
  __nv_bfloat16* o;    // [b * h, s_q, 128]
  float* lse;          // [b * h, 128, groups]
  int groups;
  int tiles;           // of a head
  long long all;       // tiles of all heads
  float low;           // least log l of a row that is right
};

VOMNI_DEV float* lse_at(const Params& p, long long bh, int row) {
  return p.lse + (bh * 128 + (row & 127)) * p.groups + (row >> 7);
}

// Whether the const-max pass's result does not stand. Its bound as it held it, in bf16.
VOMNI_DEV bool off(const Params& p, long long bh, int row) {
  const float c = __bfloat162float(__float2bfloat16_rn(p.scale * sqrtf(p.kmax2[bh] * p.qn2[bh * p.s_q + row])));
  const float log_l = *lse_at(p, bh, row) - c;
  return !(log_l >= p.low && log_l <= 44.f);  // also where it is not a number; e^44 = 2^63
}

// Byte offset of 16-byte chunk c of row r of a tile: neighbouring rows' chunks in different banks.
VOMNI_DEV uint32_t chunk_at(int r, int c) { return static_cast<uint32_t>(r * 256 + ((c ^ (r & 7)) << 4)); }

VOMNI_DEV void copy16(uint32_t dst, const void* src, bool there) {  // zeros where it is not there
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
VOMNI_DEV void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
VOMNI_DEV void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
VOMNI_DEV void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
VOMNI_DEV float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
VOMNI_DEV float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// Rows row0 + .. of head bh; writes those whose bit in `rows` is set.
VOMNI_DEV void tile_again(const Params& p, uint8_t* smem, long long bh, int row0, unsigned long long rows) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long b = bh / p.h;
  const int h = static_cast<int>(bh % p.h);
  const uint32_t base = smem_u32(smem);
  const __nv_bfloat16* kv[2] = {p.k + b * p.s_kv * p.kv_stride + h * kD, p.v + b * p.s_kv * p.kv_stride + h * kD};
  auto load = [&](int step) {
    for (int i = threadIdx.x; i < 2 * kKeys * 16; i += 32 * kWarps) {
      const int which = i / (kKeys * 16), r = i / 16 % kKeys, c = i % 16, key = step * kKeys + r;
      const bool there = key < p.s_kv;
      copy16(base + ((step & 1) * 2 + which) * kTileBytes + chunk_at(r, c),
             kv[which] + static_cast<long long>(there ? key : 0) * p.kv_stride + c * 8, there);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const int steps = (p.s_kv + kKeys - 1) / kKeys;
  load(0);

  const int mine[2] = {row0 + warp * 16 + g, row0 + warp * 16 + g + 8};  // this thread's rows
  uint32_t q[8][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool there = mine[i] < p.s_q;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(p.q + (b * p.s_q + (there ? mine[i] : 0)) * p.q_stride + h * kD);
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      q[kk][i] = there ? src[kk * 8 + t] : 0u;
      q[kk][2 + i] = there ? src[kk * 8 + 4 + t] : 0u;
    }
  }
  const float scale2 = p.scale * 1.4426950408889634f;
  float o[16][4] = {}, top[2] = {-INFINITY, -INFINITY}, sum[2] = {}, sum_b[2] = {};  // sums of P, of P as bf16: this thread's columns
  for (int j = 0; j < steps; ++j) {
    if (j + 1 < steps) {
      load(j + 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    const uint32_t sk = base + (j & 1) * 2 * kTileBytes, sv = sk + kTileBytes;
    float s[8][4] = {};
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int kk = 0; kk < 8; kk += 2) {
        uint32_t f[4];
        ldmatrix4(sk + chunk_at(n * 8 + (lane & 7), kk * 2 + (lane >> 3)), f);
        mma16816(s[n], q[kk], f[0], f[1]);
        mma16816(s[n], q[kk + 1], f[2], f[3]);
      }
    const int valid = p.s_kv - j * kKeys;
    float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (n * 8 + 2 * t + (i & 1) >= valid) s[n][i] = -INFINITY;
        most[i >> 1] = fmaxf(most[i >> 1], s[n][i]);
      }
    float from[2], shrink[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float now = fmaxf(top[i], quad_max(most[i]));
      from[i] = now == -INFINITY ? 0.f : now;  // a row whose scores are all -inf so far: its exponentials are 0
      shrink[i] = top[i] == now ? 1.f : exp2f((top[i] - from[i]) * scale2);
      top[i] = now;
      sum[i] *= shrink[i];
      sum_b[i] *= shrink[i];
    }
    uint32_t pk[8][2];  // P, two columns a word
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float p0 = exp2f((s[n][2 * i] - from[i]) * scale2), p1 = exp2f((s[n][2 * i + 1] - from[i]) * scale2);
        sum[i] += p0 + p1;
        pk[n][i] = pack_bf16x2(p0, p1);
        sum_b[i] += __uint_as_float(pk[n][i] << 16) + __uint_as_float(pk[n][i] & 0xffff0000u);
      }
#pragma unroll
    for (int n = 0; n < 16; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] *= shrink[i >> 1];
#pragma unroll
    for (int kk = 0; kk < kKeys / 16; ++kk) {
      const uint32_t a[4] = {pk[2 * kk][0], pk[2 * kk][1], pk[2 * kk + 1][0], pk[2 * kk + 1][1]};
#pragma unroll
      for (int n = 0; n < 16; n += 2) {
        uint32_t f[4];
        ldmatrix4_trans(sv + chunk_at(kk * 16 + (lane & 15), n + (lane >> 4)), f);
        mma16816(o[n], a, f[0], f[1]);
        mma16816(o[n + 1], a, f[2], f[3]);
      }
    }
    __syncthreads();  // the slot is loaded again two steps on
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float l = quad_sum(sum[i]), lb = quad_sum(sum_b[i]);
    if (!(rows >> (warp * 16 + g + 8 * i) & 1)) continue;
    const float inv = l == 0.f ? 0.f : 1.f / lb;
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.o + (bh * p.s_q + mine[i]) * kD);
#pragma unroll
    for (int n = 0; n < 16; ++n) dst[n * 4 + t] = pack_bf16x2(o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
    if (t == 0) *lse_at(p, bh, mine[i]) = l == 0.f ? -INFINITY : top[i] * p.scale + logf(l);
  }
}

// Each warp looks at the rows of one tile; the CTA then computes the tiles that have rows to do. Where none has, as with most
// inputs, that is all: 10 us for 8190 rows of 40 heads, 4 us for 77 rows of 4.
__global__ void __launch_bounds__(32 * kWarps, kCtasPerSm) attn_far_rows_kernel(const Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ unsigned long long todo[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (long long first = static_cast<long long>(blockIdx.x) * kWarps; first < p.all; first += static_cast<long long>(gridDim.x) * kWarps) {
    const long long tile = first + warp, bh = tile / p.tiles;
    const int row = static_cast<int>(tile % p.tiles) * kRows + lane;
    const bool in = tile < p.all;
    const unsigned lo = __ballot_sync(0xffffffffu, in && row < p.s_q && off(p, bh, row));
    const unsigned hi = __ballot_sync(0xffffffffu, in && row + 32 < p.s_q && off(p, bh, row + 32));
    if (lane == 0) todo[warp] = static_cast<unsigned long long>(hi) << 32 | lo;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w)
      if (todo[w]) tile_again(p, smem, (first + w) / p.tiles, static_cast<int>((first + w) % p.tiles) * kRows, todo[w]);
    __syncthreads();
  }
}

}  // namespace afwd
}  // namespace vomni

using namespace vomni;

extern "C" int vomni_attention_fwd(const void* q, const void* k, const void* v, void* out, float* lse, int b, int s_q, int s_kv, int h,
                                   int d, long long q_stride, long long kv_stride, float softmax_scale, void* workspace,
                                   size_t workspace_bytes, vomni_stream_t stream) {
  if (!v || !out || !lse) return VOMNI_EINVAL;
  if ((reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(out)) & 15 || reinterpret_cast<uintptr_t>(lse) & 3) return VOMNI_EALIGN;
  if (!(softmax_scale >= 1e-20f && softmax_scale <= 1e20f)) return VOMNI_EINVAL;
  int rc = vomni_cm_attention_cross(q, k, v, out, lse, b, s_q, s_kv, h, d, q_stride, kv_stride, softmax_scale, VOMNI_CM_LSE, workspace,
                                    workspace_bytes, stream);
  if (rc) return rc;
  using namespace afwd;
  Params p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.q_stride = q_stride ? q_stride : static_cast<long long>(h) * d;
  p.kv_stride = kv_stride ? kv_stride : static_cast<long long>(h) * d;
  p.s_q = s_q;
  p.s_kv = s_kv;
  p.h = h;
  p.scale = softmax_scale;
  // the norms, where vomni_cm_attention_cross left them
  p.qn2 = static_cast<const float*>(workspace);
  p.kmax2 = reinterpret_cast<const float*>(static_cast<const uint8_t*>(workspace) +
                                           align_up(static_cast<size_t>(b) * h * s_q * sizeof(float), 256));
  p.o = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.groups = (s_q + 127) / 128;
  p.tiles = (s_q + kRows - 1) / kRows;
  p.all = static_cast<long long>(p.tiles) * b * h;
  p.low = std::log(static_cast<float>(s_kv)) - 102.f * 0.6931472f;
  rc = ensure_max_smem(attn_far_rows_kernel, kSmemBytes);
  if (rc) return rc;
  const long long need = (p.all + kWarps - 1) / kWarps, most = static_cast<long long>(num_sms()) * kCtasPerSm;
  attn_far_rows_kernel<<<static_cast<unsigned>(std::min(need, most)), 32 * kWarps, kSmemBytes, reinterpret_cast<cudaStream_t>(stream)>>>(p);
  VOMNI_CUDA_TRY(cudaGetLastError());
  return VOMNI_OK;
}
