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
// HBM-bound: 4 rows of 2H bytes a token forward, 6 backward, each read or written once. A thread owns
// 8 adjacent columns and keeps their values of a row in registers between the reductions.
// The backward pass is persistent, so that a thread's
// column sums stay in its registers over all rows of its CTA; the CTAs' sums go to a workspace
// and are added in a fixed order by a second kernel (no atomics: the same call gives the same bits).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "host_util.h"

namespace vomni {
namespace sandwich {

constexpr int kMaxH = 8192;  // 8 columns a thread, 1024 threads
constexpr int kLayer = 0, kNone = 2;  // 1: RMSNorm
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
  long long rows, rows_per_mod;
  long long gate_step, mul_step, add_step;  // H where per modulation row, else 0
  int H, post, norm;
  float eps, inv_h;
  __nv_bfloat16* out0;  // forward: residual_out; backward: dx
  __nv_bfloat16* out1;  // forward: out; backward: dresidual
  float* parts;         // backward: [n_mod][gridDim.x][3][H]
};

VOMNI_DEV void unpack8(const uint4& w, float (&v)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(u[i] << 16);
    v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
VOMNI_DEV uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
VOMNI_DEV void load8(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// Sums N values over the threads of a row: one warp (kWarpRow), or the whole CTA through shared memory.
// Every thread ends with the same sums, added in the same order. `turn` alternates between two
// buffers: a buffer is written again only after a barrier that follows its last read.
template <int N, bool kWarpRow>
VOMNI_DEV void row_sum(float (&v)[N], float (*buf)[32 * 2], int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (kWarpRow) return;
  static_assert(N <= 2, "buffer holds two values per warp");
  float* b = buf[turn];
  turn ^= 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) b[i * 32 + warp] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane < warps ? b[i * 32 + lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
}

// v -> its normalised values; returns 1 / deviation. Two passes (mean, then squared deviations) in fp32.
template <bool kWarpRow>
VOMNI_DEV float normalise(float (&v)[8], int kind, bool in, const Params& p, float (*buf)[64], int& turn) {
  if (kind == kNone) return 1.f;
  float s[1];
  if (kind == kLayer) {
    s[0] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    row_sum<1, kWarpRow>(s, buf, turn);
    const float mean = s[0] * p.inv_h;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = in ? v[i] - mean : 0.f;
  }
  s[0] = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s[0] = fmaf(v[i], v[i], s[0]);
  row_sum<1, kWarpRow>(s, buf, turn);
  const float rstd = rsqrtf(s[0] * p.inv_h + p.eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= rstd;
  return rstd;
}

// d -> the gradient behind normalise(): rstd (d - [mean d] - hat mean(d hat)).
template <bool kWarpRow>
VOMNI_DEV void normalise_grad(float (&d)[8], const float (&hat)[8], float rstd, int kind, const Params& p,
                              float (*buf)[64], int& turn) {
  if (kind == kNone) return;
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    s[0] += d[i];
    s[1] = fmaf(d[i], hat[i], s[1]);
  }
  row_sum<2, kWarpRow>(s, buf, turn);
  const float m0 = kind == kLayer ? s[0] * p.inv_h : 0.f, m1 = s[1] * p.inv_h;
#pragma unroll
  for (int i = 0; i < 8; ++i) d[i] = rstd * (d[i] - m0 - hat[i] * m1);
}

// A row per warp (kWarpRow: H <= 256, blockDim.y rows a CTA) or per CTA.
template <int kMaxThreads, bool kWarpRow>
__global__ void __launch_bounds__(kMaxThreads) sandwich_fwd_kernel(const Params p) {
  __shared__ float buf[2][64];
  int turn = 0;
  const int c = threadIdx.x * 8;
  const bool in = c < p.H;
  const long long step = static_cast<long long>(gridDim.x) * blockDim.y;
  for (long long row = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y; row < p.rows; row += step) {
    const long long at = row * p.H + c;
    const long long mod = row / p.rows_per_mod;
    float r[8] = {};
    if (in) unpack8(__ldcs(reinterpret_cast<const uint4*>(p.residual + at)), r);
    if (p.x) {
      float y[8] = {};
      if (in) unpack8(__ldcs(reinterpret_cast<const uint4*>(p.x + at)), y);
      normalise<kWarpRow>(y, p.post, in, p, buf, turn);
      if (in) {
        float w[8];
        if (p.post_w) {
          load8(p.post_w + c, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] *= w[i];
        }
        if (p.gate) {
          load8(p.gate + mod * p.gate_step + c, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) r[i] = fmaf(w[i], y[i], r[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) r[i] += y[i];
        }
        __stcs(reinterpret_cast<uint4*>(p.out0 + at), pack8(r));
      }
    }
    normalise<kWarpRow>(r, p.norm, in, p, buf, turn);
    if (in) {
      float m[8], a[8];
      if (p.mul) {
        load8(p.mul + mod * p.mul_step + c, m);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] *= m[i];
      }
      if (p.add) {
        load8(p.add + mod * p.add_step + c, a);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] += a[i];
      }
      __stcs(reinterpret_cast<uint4*>(p.out1 + at), pack8(r));
    }
  }
}

// gridDim.y modulation rows; the rows of one are dealt to gridDim.x CTAs (x blockDim.y warps).
template <int kMaxThreads, bool kWarpRow>
__global__ void __launch_bounds__(kMaxThreads) sandwich_bwd_kernel(const Params p) {
  __shared__ float buf[2][64];
  int turn = 0;
  const int c = threadIdx.x * 8;
  const bool in = c < p.H;
  const long long mod = blockIdx.y;
  const long long end = (mod + 1) * p.rows_per_mod;
  const int lanes = gridDim.x * blockDim.y, lane = blockIdx.x * blockDim.y + threadIdx.y;
  float sum_a[8] = {}, sum_m[8] = {}, sum_d[8] = {};
  for (long long row = mod * p.rows_per_mod + lane; row < end; row += lanes) {
    const long long at = row * p.H + c;
    float dr[8] = {}, n[8] = {}, w[8];
    if (in && p.d_res) unpack8(__ldcs(reinterpret_cast<const uint4*>(p.d_res + at)), dr);
    if (p.d_out) {
      float g[8] = {};
      if (in) {
        unpack8(__ldcs(reinterpret_cast<const uint4*>(p.d_out + at)), g);
        unpack8(__ldcs(reinterpret_cast<const uint4*>(p.residual + at)), n);
      }
      const float rstd = normalise<kWarpRow>(n, p.norm, in, p, buf, turn);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum_m[i] = fmaf(g[i], n[i], sum_m[i]);
        sum_d[i] += g[i];
      }
      if (p.mul && in) {
        load8(p.mul + mod * p.mul_step + c, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] *= w[i];
      }
      normalise_grad<kWarpRow>(g, n, rstd, p.norm, p, buf, turn);
#pragma unroll
      for (int i = 0; i < 8; ++i) dr[i] = in ? dr[i] + g[i] : 0.f;
    }
    if (in) __stcs(reinterpret_cast<uint4*>(p.out1 + at), pack8(dr));
    if (p.x) {
      float y[8] = {};
      if (in) unpack8(__ldcs(reinterpret_cast<const uint4*>(p.x + at)), y);
      const float rstd = normalise<kWarpRow>(y, p.post, in, p, buf, turn);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum_a[i] = fmaf(dr[i], y[i], sum_a[i]);
      if (in && p.gate) {
        load8(p.gate + mod * p.gate_step + c, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) dr[i] *= w[i];
      }
      if (in && p.post_w) {
        load8(p.post_w + c, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) dr[i] *= w[i];
      }
      normalise_grad<kWarpRow>(dr, y, rstd, p.post, p, buf, turn);
      if (in) __stcs(reinterpret_cast<uint4*>(p.out0 + at), pack8(dr));
    }
  }
  if (!in) return;
  float* part = p.parts + (mod * lanes + lane) * 3 * p.H + c;
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    const float(&s)[8] = q == 0 ? sum_a : q == 1 ? sum_m : sum_d;
    reinterpret_cast<float4*>(part + static_cast<size_t>(q) * p.H)[0] = make_float4(s[0], s[1], s[2], s[3]);
    reinterpret_cast<float4*>(part + static_cast<size_t>(q) * p.H)[1] = make_float4(s[4], s[5], s[6], s[7]);
  }
}

struct SumParams {
  const float* parts;  // [n_mod][lanes][3][H]
  const float* gate;
  const float* post_w;
  long long gate_step;
  int H, lanes, n_mod, per;  // per: kPer* flags
  float *dgate, *dpost_w, *dmul, *dadd;
};

// 32 columns x 8 lanes a CTA; blockIdx.y: A, M or D. Sums each modulation row's parts in the order
// lane, lane + 8, ..., then the 8 lanes in order, and forms the outputs; those shared by the
// modulation rows are added over them in order.
__global__ void __launch_bounds__(256) sandwich_sum_kernel(const SumParams p) {
  __shared__ float red[8][32];
  const int col = blockIdx.x * 32 + threadIdx.x, q = blockIdx.y;
  const bool in = col < p.H;
  float shared_out = 0.f, dw = 0.f;
  float* out = q == 0 ? p.dgate : q == 1 ? p.dmul : p.dadd;
  const bool per = p.per & (q == 0 ? kPerGate : q == 1 ? kPerMul : kPerAdd);
  if (!out && !(q == 0 && p.dpost_w)) return;
  for (int mod = 0; mod < p.n_mod; ++mod) {
    float s = 0.f;
    if (in)
      for (int l = threadIdx.y; l < p.lanes; l += 8)
        s += p.parts[((static_cast<long long>(mod) * p.lanes + l) * 3 + q) * p.H + col];
    red[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && in) {
      float t = 0.f;
#pragma unroll
      for (int l = 0; l < 8; ++l) t += red[l][threadIdx.x];
      if (q == 0 && p.dpost_w) dw = fmaf(t, p.gate ? p.gate[mod * p.gate_step + col] : 1.f, dw);
      if (q == 0 && p.post_w) t *= p.post_w[col];
      if (per) {
        if (out) out[static_cast<long long>(mod) * p.H + col] = t;
      } else {
        shared_out += t;
      }
    }
    __syncthreads();
  }
  if (threadIdx.y == 0 && in) {
    if (out && !per) out[col] = shared_out;
    if (q == 0 && p.dpost_w) p.dpost_w[col] = dw;
  }
}

// Threads of a row (a multiple of 32) and rows per CTA.
struct Shape {
  int tx, ty;
};
Shape shape_of(int h) {
  const int chunks = h / 8;
  if (chunks <= 32) return {32, 4};
  return {(chunks + 31) / 32 * 32, 1};
}
// Lanes (CTAs x rows per CTA) that share a modulation row's tokens in the backward pass: enough to fill
// the device once over all modulation rows.
int bwd_blocks(long long rows_per_mod, long long n_mod, const Shape& sh) {
  const int per_sm = 1024 / (sh.tx * sh.ty) > 0 ? 1024 / (sh.tx * sh.ty) : 1;
  const long long cap = (static_cast<long long>(num_sms()) * per_sm + n_mod - 1) / n_mod;
  const long long need = (rows_per_mod + sh.ty - 1) / sh.ty;
  return static_cast<int>(need < cap ? need : cap);
}

int check(long long rows, int h, long long rows_per_mod, int post, int norm) {
  if (rows <= 0 || rows > 0x7fffffffLL || h <= 0 || h > kMaxH || h % 8) return VOMNI_EBADSHAPE;
  if (rows_per_mod <= 0 || rows % rows_per_mod) return VOMNI_EBADSHAPE;
  if (post < 0 || post > 2 || norm < 0 || norm > 2) return VOMNI_EINVAL;
  return VOMNI_OK;
}
bool misaligned(const void* a, const void* b = nullptr, const void* c = nullptr, const void* d = nullptr) {
  return (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) |
          reinterpret_cast<uintptr_t>(d)) & 15;
}
void fill(Params& p, const void* x, const void* residual, const float* gate, const float* post_w, const float* mul,
          const float* add, long long rows, int h, long long rows_per_mod, int per, float eps, int post, int norm) {
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.residual = static_cast<const __nv_bfloat16*>(residual);
  p.gate = gate;
  p.post_w = post_w;
  p.mul = mul;
  p.add = add;
  p.rows = rows;
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
  if (!x && (gate || post_weight)) return VOMNI_EINVAL;
  int rc = check(rows, h, rows_per_mod, post_norm, norm_type);
  if (rc) return rc;
  if (misaligned(x, residual, residual_out, out) || misaligned(gate, post_weight, mul, add)) return VOMNI_EALIGN;
  rc = require_sm100();
  if (rc) return rc;
  Params p = {};
  fill(p, x, residual, gate, post_weight, mul, add, rows, h, rows_per_mod, per_mod, eps, post_norm, norm_type);
  p.out0 = static_cast<__nv_bfloat16*>(residual_out);
  p.out1 = static_cast<__nv_bfloat16*>(out);
  const Shape sh = shape_of(h);
  const dim3 block(sh.tx, sh.ty);
  const unsigned grid = static_cast<unsigned>((rows + sh.ty - 1) / sh.ty);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (sh.tx == 32)
    sandwich_fwd_kernel<128, true><<<grid, block, 0, st>>>(p);
  else if (sh.tx <= 512)
    sandwich_fwd_kernel<512, false><<<grid, block, 0, st>>>(p);
  else
    sandwich_fwd_kernel<1024, false><<<grid, block, 0, st>>>(p);
  VOMNI_CUDA_TRY(cudaGetLastError());
  return VOMNI_OK;
}

extern "C" size_t vomni_sandwich_norm_workspace_bytes(long long rows, int h, long long rows_per_mod) {
  using namespace sandwich;
  if (check(rows, h, rows_per_mod, 0, 0)) return 0;
  const Shape sh = shape_of(h);
  const long long n_mod = rows / rows_per_mod;
  return static_cast<size_t>(n_mod) * bwd_blocks(rows_per_mod, n_mod, sh) * sh.ty * 3 * h * sizeof(float);
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
  int rc = check(rows, h, rows_per_mod, post_norm, norm_type);
  if (rc) return rc;
  const long long n_mod = rows / rows_per_mod;
  if (n_mod > 65535) return VOMNI_EBADSHAPE;
  if (workspace_bytes < vomni_sandwich_norm_workspace_bytes(rows, h, rows_per_mod)) return VOMNI_EWORKSPACE;
  if (misaligned(x, residual_out, grad_residual_out, grad_out) || misaligned(gate, post_weight, mul, workspace) ||
      misaligned(dx, dresidual))
    return VOMNI_EALIGN;
  rc = require_sm100();
  if (rc) return rc;
  Params p = {};
  fill(p, x, residual_out, gate, post_weight, mul, nullptr, rows, h, rows_per_mod, per_mod, eps, post_norm, norm_type);
  p.d_res = static_cast<const __nv_bfloat16*>(grad_residual_out);
  p.d_out = static_cast<const __nv_bfloat16*>(grad_out);
  p.out0 = static_cast<__nv_bfloat16*>(dx);
  p.out1 = static_cast<__nv_bfloat16*>(dresidual);
  p.parts = static_cast<float*>(workspace);
  const Shape sh = shape_of(h);
  const dim3 block(sh.tx, sh.ty);
  const dim3 grid(bwd_blocks(rows_per_mod, n_mod, sh), static_cast<unsigned>(n_mod));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (sh.tx == 32)
    sandwich_bwd_kernel<128, true><<<grid, block, 0, st>>>(p);
  else if (sh.tx <= 512)
    sandwich_bwd_kernel<512, false><<<grid, block, 0, st>>>(p);
  else
    sandwich_bwd_kernel<1024, false><<<grid, block, 0, st>>>(p);
  VOMNI_CUDA_TRY(cudaGetLastError());
  if (!dgate && !dpost_weight && !dmul && !dadd) return VOMNI_OK;
  SumParams s = {};
  s.parts = p.parts;
  s.gate = gate;
  s.post_w = post_weight;
  s.gate_step = p.gate_step;
  s.H = h;
  s.lanes = static_cast<int>(grid.x) * sh.ty;
  s.n_mod = static_cast<int>(n_mod);
  s.per = per_mod;
  s.dgate = dgate;
  s.dpost_w = dpost_weight;
  s.dmul = dmul;
  s.dadd = dadd;
  sandwich_sum_kernel<<<dim3((h + 31) / 32, 3), dim3(32, 8), 0, st>>>(s);
  VOMNI_CUDA_TRY(cudaGetLastError());
  return VOMNI_OK;
}
