// Rotary positions with several axes (frame, row, column of a video; row, column of an image), and
// their gradient, for query and key heads in one launch.
//
// A head of d values is d / 2 pairs, split among the axes: axis a owns n_a / 2 consecutive pairs
// (sum n_a = d), its pair i turning by
//     angle = position[a] * theta^(-2 i / n_a),  (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin),
// with (x1, x2) = (x[2p], x[2p+1]) (interleaved) or (x[p], x[p + d/2]) (rotate-half). The gradient is
// the rotation by the negative angle. With axes (44, 42, 42) and interleaved pairs this is
// WanRotaryPosEmbed + apply_rotary_emb_wan (vllm_omni_neuron/diffusion/layers/rope.py:8-114) without
// their per-token tables.
//
// Angles: the frequency is kept as turns per position (theta^(-2i/n) / 2 pi) in fp64, the product
// with the position is reduced to [-1/2, 1/2] turns in fp64 and only then rounded to fp32, so a
// far position costs no accuracy up to some 10^8 (2^-24 relative of the reduced angle; the fp64 product is off
// by 2^-52 of the turns; an fp32 product at position 10^6 would be off by 0.06 rad).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "host_util.h"

namespace vomni {
namespace rotary {

constexpr int kMaxDim = 256;
constexpr int kMaxAxes = 4;
constexpr int kGroup = 8;  // pairs per thread and head: 16 values, two 16-byte loads in 16-bit types
constexpr int kThreads = 128;

struct Tensor {
  const void* x;
  void* y;  // dense [b, s, heads, d]
  int heads;
  long long row_stride, batch_stride;  // of x, in elements
};

struct Params {
  Tensor t[2];
  long long tokens;  // b * s
  int s, d, n_axes;
  int per;          // tokens of a CTA
  int head_blocks;  // CTAs that share their heads
  const void* pos;  // [s, n_axes] or [b, s, n_axes]
  int pos_type;     // 0 int32, 1 int64, 2 fp32
  int pos_batch;    // positions differ per batch element
  int half;         // rotate-half pairs
  float sign;       // -1: the inverse rotation (the gradient)
  unsigned char axis[kMaxDim / 2];
  double turns[kMaxDim / 2];  // turns per unit of position
};

// Eight adjacent values as they come from memory, and as floats.
template <typename T>
struct Io {  // 16-bit types
  static constexpr int kAhead = 4;  // heads whose values a thread has in flight
  using Raw = uint4;
  static VOMNI_DEV Raw load8(const T* p) { return __ldcs(reinterpret_cast<const uint4*>(p)); }
  static VOMNI_DEV void unpack(const Raw& w, float (&v)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
  static VOMNI_DEV void store8(T* p, const float (&v)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        u[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(u[0], u[1], u[2], u[3]));
  }
};
template <>
struct Io<float> {
  static constexpr int kAhead = 2;
  struct Raw {
    float4 a, b;
  };
  static VOMNI_DEV Raw load8(const float* p) {
    return {__ldcs(reinterpret_cast<const float4*>(p)), __ldcs(reinterpret_cast<const float4*>(p) + 1)};
  }
  static VOMNI_DEV void unpack(const Raw& w, float (&v)[8]) {
    v[0] = w.a.x; v[1] = w.a.y; v[2] = w.a.z; v[3] = w.a.w; v[4] = w.b.x; v[5] = w.b.y; v[6] = w.b.z; v[7] = w.b.w;
  }
  static VOMNI_DEV void store8(float* p, const float (&v)[8]) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
    __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(v[4], v[5], v[6], v[7]));
  }
};

// A CTA takes `p.per` tokens (and, of few tokens, a share of their heads). Each pair's cosine and sine is formed once, by
// one thread, into shared memory; then thread t works on pair group t % (d / 16) of heads t / (d / 16), ...; d / 16 need not
// divide kThreads: the threads past the last whole head idle. A thread has kAhead heads' values in flight, the first of them
// while the table is made. HBM-bound: every value is read and written once.
// Measured, 32760 tokens of 80 heads of 128 in bf16 (1.34 GB): 212 us, 6.3 TB/s, 0.97 of the measured copy. With every
// thread forming the eight angles it uses (32 times over at 80 heads) 351 us; first loads after the table 281 us instead of
// 267; sixteen adjacent values a thread and the table by pairs, which filled the L1's data pipe with bank conflicts and half
// used lines (83 % of its wavefronts), 253 us.
template <typename T>
__global__ void __launch_bounds__(kThreads, 6) rotary_kernel(const __grid_constant__ Params p) {
  __shared__ __align__(16) float2 table[kThreads];  // [per][d / 2] (cosine, sine)
  const int groups = p.d / (2 * kGroup), pairs = p.d / 2;
  const int lanes = kThreads / groups;  // heads in flight
  const int g = threadIdx.x % groups, lane = threadIdx.x / groups;
  const long long token0 = static_cast<long long>(blockIdx.x / p.head_blocks) * p.per;
  const int share = blockIdx.x % p.head_blocks;
  const int count = static_cast<int>(min(static_cast<long long>(p.per), p.tokens - token0));

  const long long b0 = token0 / p.s;
  const int s0 = static_cast<int>(token0 - b0 * p.s);

  // values of the group: 8 of each half of the head, so that neighbouring threads load neighbouring 16 bytes. They are pairs
  // 8 g .. 8 g + 7 (rotate-half), or 4 g .. 4 g + 3 and the same behind the middle (interleaved).
  const int o1 = g * 8, o2 = o1 + p.d / 2;
  const int all = p.t[0].heads + p.t[1].heads, step = p.head_blocks * lanes;
  int k = lane < lanes ? 0 : count, h = share * lanes + lane;  // token of the CTA, head over both tensors
  constexpr int kAhead = Io<T>::kAhead;
  typename Io<T>::Raw ra[kAhead], rb[kAhead];
  T* y[kAhead];
  int tok[kAhead];
  auto fetch = [&] {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      while (h >= all) {
        h -= all;
        ++k;
      }
      y[u] = nullptr;
      tok[u] = k;
      if (k < count) {
        long long bi = b0;
        int si = s0 + k;
        while (si >= p.s) {
          si -= p.s;
          ++bi;
        }
        const int which = h >= p.t[0].heads;
        const Tensor& t = p.t[which];
        const int hh = which ? h - p.t[0].heads : h;
        const T* x = static_cast<const T*>(t.x) + bi * t.batch_stride + si * t.row_stride + static_cast<long long>(hh) * p.d;
        y[u] = static_cast<T*>(t.y) + ((token0 + k) * t.heads + hh) * p.d;
        ra[u] = Io<T>::load8(x + o1);
        rb[u] = Io<T>::load8(x + o2);
      }
      h += step;
    }
  };
  fetch();  // under way while the table is made

  if (threadIdx.x < count * pairs) {
    const int pair = threadIdx.x % pairs, tk = threadIdx.x / pairs;
    const long long token = p.pos_batch ? token0 + tk : (s0 + tk) % p.s;
    const long long at = token * p.n_axes + p.axis[pair];
    const double pos = p.pos_type == 0   ? static_cast<double>(static_cast<const int*>(p.pos)[at])
                       : p.pos_type == 1 ? static_cast<double>(static_cast<const long long*>(p.pos)[at])
                                         : static_cast<double>(static_cast<const float*>(p.pos)[at]);
    double t = pos * p.turns[pair];
    t -= rint(t);
    float sn, c;
    sincospif(2.f * static_cast<float>(t), &sn, &c);
    // the four float4 (two pairs each) that a group reads lie `groups` apart: a quarter-warp reads 128 adjacent bytes
    const int behind = !p.half && pair >= pairs / 2, q = behind ? pair - pairs / 2 : pair;
    const int owner = p.half ? q / 8 : q / 4, i = p.half ? q % 8 / 2 : q % 4 / 2 + 2 * behind;
    table[tk * pairs + (i * groups + owner) * 2 + (pair & 1)] = make_float2(c, sn * p.sign);
  }
  __syncthreads();

  while (y[0]) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (!y[u]) break;
      float a[8], b[8], c[kGroup], sn[kGroup];
      Io<T>::unpack(ra[u], a);
      Io<T>::unpack(rb[u], b);
      const float4* cs = reinterpret_cast<const float4*>(table + tok[u] * pairs) + g;
#pragma unroll
      for (int i = 0; i < kGroup / 2; ++i) {
        const float4 w = cs[i * groups];
        c[2 * i] = w.x; sn[2 * i] = w.y; c[2 * i + 1] = w.z; sn[2 * i + 1] = w.w;
      }
      if (p.half) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x1 = a[i], x2 = b[i];
          a[i] = x1 * c[i] - x2 * sn[i];
          b[i] = x2 * c[i] + x1 * sn[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x1 = a[2 * i], x2 = a[2 * i + 1], z1 = b[2 * i], z2 = b[2 * i + 1];
          a[2 * i] = x1 * c[i] - x2 * sn[i];
          a[2 * i + 1] = x2 * c[i] + x1 * sn[i];
          b[2 * i] = z1 * c[4 + i] - z2 * sn[4 + i];
          b[2 * i + 1] = z2 * c[4 + i] + z1 * sn[4 + i];
        }
      }
      Io<T>::store8(y[u] + o1, a);
      Io<T>::store8(y[u] + o2, b);
    }
    fetch();
  }
}

int check_tensor(const void* x, const void* y, int heads, long long row_stride, long long batch_stride, int b, int s,
                 int d, int esize) {
  if (heads < 0 || heads > (1 << 20)) return VOMNI_EBADSHAPE;
  if (heads == 0) return VOMNI_OK;
  if (!x || !y) return VOMNI_EINVAL;
  if (s > 1 && row_stride < static_cast<long long>(heads) * d) return VOMNI_EBADSHAPE;
  if (b > 1 && batch_stride < 0) return VOMNI_EBADSHAPE;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) return VOMNI_EALIGN;
  if ((row_stride * esize) % 16 || (batch_stride * esize) % 16) return VOMNI_EALIGN;
  return VOMNI_OK;
}

// The pairs' axes and frequencies. A thread keeps the last ones it formed: a model asks for the same every time, and the
// powers take some microseconds.
struct Frequencies {
  int d = 0, n_axes = 0, dims[kMaxAxes] = {};
  double theta = 0.0;
  unsigned char axis[kMaxDim / 2];
  double turns[kMaxDim / 2];
};
int frequencies(Params& p, int n_axes, const int* dims, int d, double theta) {
  static thread_local Frequencies f;
  bool same = f.d == d && f.n_axes == n_axes && f.theta == theta;
  for (int a = 0; same && a < n_axes; ++a) same = f.dims[a] == dims[a];
  if (!same) {
    f.d = 0;  // until it is whole
    int pair = 0;
    for (int a = 0; a < n_axes; ++a) {
      if (dims[a] <= 0 || dims[a] % 2 || pair + dims[a] / 2 > d / 2) return VOMNI_EBADSHAPE;
      for (int i = 0; i < dims[a] / 2; ++i, ++pair) {
        f.axis[pair] = static_cast<unsigned char>(a);
        f.turns[pair] = std::pow(theta, -2.0 * i / dims[a]) / 6.283185307179586476925286766559;
      }
      f.dims[a] = dims[a];
    }
    if (pair != d / 2) return VOMNI_EBADSHAPE;
    f.n_axes = n_axes;
    f.theta = theta;
    f.d = d;
  }
  std::copy(f.axis, f.axis + d / 2, p.axis);
  std::copy(f.turns, f.turns + d / 2, p.turns);
  return VOMNI_OK;
}

}  // namespace rotary
}  // namespace vomni

using namespace vomni;

extern "C" int vomni_rotary_axes(const void* q, void* q_out, int q_heads, long long q_row_stride,
                                 long long q_batch_stride, const void* k, void* k_out, int k_heads,
                                 long long k_row_stride, long long k_batch_stride, int b, int s, int d,
                                 const void* positions, int pos_type, int pos_per_batch, int n_axes,
                                 const int* axes_dims, double theta, int pairing, int inverse, int dtype,
                                 vomni_stream_t stream) {
  if (!positions || !axes_dims) return VOMNI_EINVAL;
  if (pos_type < 0 || pos_type > 2 || pairing < 0 || pairing > 1 || dtype < 0 || dtype > 2) return VOMNI_EINVAL;
  if (!(theta > 0.0) || !std::isfinite(theta)) return VOMNI_EINVAL;
  if (b <= 0 || s <= 0 || d <= 0 || d > rotary::kMaxDim || d % 16) return VOMNI_EBADSHAPE;
  if (n_axes < 1 || n_axes > rotary::kMaxAxes) return VOMNI_EBADSHAPE;
  const int esize = dtype == 2 ? 4 : 2;
  int rc = rotary::check_tensor(q, q_out, q_heads, q_row_stride, q_batch_stride, b, s, d, esize);
  if (rc) return rc;
  rc = rotary::check_tensor(k, k_out, k_heads, k_row_stride, k_batch_stride, b, s, d, esize);
  if (rc) return rc;
  if (q_heads + k_heads == 0) return VOMNI_EBADSHAPE;
  if (reinterpret_cast<uintptr_t>(positions) & (pos_type == 1 ? 7 : 3)) return VOMNI_EALIGN;
  rotary::Params p;
  rc = rotary::frequencies(p, n_axes, axes_dims, d, theta);
  if (rc) return rc;
  rc = require_sm100();
  if (rc) return rc;
  p.t[0] = {q, q_out, q_heads, q_row_stride, q_batch_stride};
  p.t[1] = {k, k_out, k_heads, k_row_stride, k_batch_stride};
  p.tokens = static_cast<long long>(b) * s;
  p.s = s;
  p.d = d;
  p.n_axes = n_axes;
  p.pos = positions;
  p.pos_type = pos_type;
  p.pos_batch = pos_per_batch != 0;
  p.half = pairing;
  p.sign = inverse ? -1.f : 1.f;
  // As many tokens a CTA as its threads have pairs for; where that leaves SMs idle, one, and its heads shared among CTAs
  // until every thread has one group.
  const int lanes = rotary::kThreads / (d / (2 * rotary::kGroup));
  const long long slots = static_cast<long long>(num_sms()) * 4;
  p.per = rotary::kThreads / (d / 2) < 8 ? rotary::kThreads / (d / 2) : 8;
  while (p.per > 1 && (p.tokens + p.per - 1) / p.per < slots) p.per /= 2;
  const int most = (q_heads + k_heads + lanes - 1) / lanes;
  const long long want = (slots + p.tokens - 1) / p.tokens;
  p.head_blocks = p.per > 1 ? 1 : static_cast<int>(want < most ? want : most);
  const long long blocks = (p.tokens + p.per - 1) / p.per * p.head_blocks;
  if (blocks > 0x7fffffffll) return VOMNI_EBADSHAPE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == 0)
    rotary::rotary_kernel<__nv_bfloat16><<<static_cast<unsigned>(blocks), rotary::kThreads, 0, st>>>(p);
  else if (dtype == 1)
    rotary::rotary_kernel<__half><<<static_cast<unsigned>(blocks), rotary::kThreads, 0, st>>>(p);
  else
    rotary::rotary_kernel<float><<<static_cast<unsigned>(blocks), rotary::kThreads, 0, st>>>(p);
  VOMNI_CUDA_TRY(cudaGetLastError());
  return VOMNI_OK;
}
