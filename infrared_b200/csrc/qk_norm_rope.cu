// RMS norm of every query and key head with the rotary embedding, one pass:
//   y = x * rsqrt(mean(x^2) + eps) * w        (over the head's D elements)
//   out[d]       = y[d] * cos[d]       - y[d + D/2] * sin[d]          d <  D/2
//   out[d + D/2] = y[d + D/2] * cos[d + D/2] + y[d] * sin[d + D/2]
// in fp32 with one rounding at the end (the values may differ in the last
// place from rotating a row that was rounded after its norm).
//
// Bound by HBM: each row is read and written once; cos, sin and the weights
// stay in registers while a group of D / 8 lanes walks heads of one token.
// A lane holds elements 4 i .. 4 i + 3 of both halves, so a rotation needs no
// other lane and the group reads two contiguous pieces of D elements' half.
#include "common.cuh"
#include "kernels.h"

namespace irb {

namespace {

constexpr int kNormThreads = 256;

template <typename T, bool VEC>
__device__ __forceinline__ float4 load_row4(const T* p) {
  if constexpr (!VEC) {
    return make_float4(DT<T>::to_f(p[0]), DT<T>::to_f(p[1]), DT<T>::to_f(p[2]),
                       DT<T>::to_f(p[3]));
  } else if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
    return make_float4(a.x, a.y, b.x, b.y);
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_row4(T* p, float4 v) {
  if constexpr (!VEC) {
    p[0] = DT<T>::from_f(v.x);
    p[1] = DT<T>::from_f(v.y);
    p[2] = DT<T>::from_f(v.z);
    p[3] = DT<T>::from_f(v.w);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = v;
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
  }
}

// Heads of one token by a group of D / 8 lanes, kBatch at a time: their loads
// are all in flight before the first sum (32768 rows of 28 + 4 heads of 128,
// bf16: 99 us = 5.75 TB/s; batches of 2 and 8 take 102 and 121, one by one 119).
constexpr int kBatch = 4;

template <typename T, int D, bool VEC>
__device__ __forceinline__ void norm_heads(const T* src, T* dst, int h0, int h1, float4 w0,
                                           float4 w1, float4 c0, float4 c1, float4 s0, float4 s1,
                                           float eps, int lo, int hi, bool live) {
  for (int h = h0; h < h1; h += kBatch) {
    float4 x[kBatch], y[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int hh = min(h + i, h1 - 1);
      x[i] = load_row4<T, VEC>(src + hh * D + lo);
      y[i] = load_row4<T, VEC>(src + hh * D + hi);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      float ss = x[i].x * x[i].x + x[i].y * x[i].y + x[i].z * x[i].z + x[i].w * x[i].w +
                 y[i].x * y[i].x + y[i].y * y[i].y + y[i].z * y[i].z + y[i].w * y[i].w;
#pragma unroll
      for (int o = D / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss * (1.f / D) + eps);
      const float4 u = make_float4(x[i].x * r * w0.x, x[i].y * r * w0.y, x[i].z * r * w0.z,
                                   x[i].w * r * w0.w);
      const float4 v = make_float4(y[i].x * r * w1.x, y[i].y * r * w1.y, y[i].z * r * w1.z,
                                   y[i].w * r * w1.w);
      if (live && h + i < h1) {
        T* o = dst + (h + i) * D;
        store_row4<T, VEC>(o + lo, make_float4(u.x * c0.x - v.x * s0.x, u.y * c0.y - v.y * s0.y,
                                               u.z * c0.z - v.z * s0.z, u.w * c0.w - v.w * s0.w));
        store_row4<T, VEC>(o + hi, make_float4(v.x * c1.x + u.x * s1.x, v.y * c1.y + u.y * s1.y,
                                               v.z * c1.z + u.z * s1.z, v.w * c1.w + u.w * s1.w));
      }
    }
  }
}

// Grid: tokens (x) and pieces of hpg heads (y); heads 0 .. H-1 are the
// query's, the rest the key's.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kNormThreads) qk_norm_rope_kernel(const NormRopeArgs a) {
  constexpr int LPR = D / 8;
  const int lane = threadIdx.x % LPR;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kNormThreads / LPR) + threadIdx.x / LPR;
  const bool live = t < a.n;
  const int64_t tok = live ? t : a.n - 1;  // idle groups follow along for the shuffles
  const int lo = lane * 4, hi = D / 2 + lane * 4;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float* cr = a.cos + tok * a.rope_stride;
  const float* sr = a.sin + tok * a.rope_stride;
  const float4 c0 = load_row4<float, VEC>(cr + lo), c1 = load_row4<float, VEC>(cr + hi);
  const float4 s0 = load_row4<float, VEC>(sr + lo), s1 = load_row4<float, VEC>(sr + hi);
  const float4 one = make_float4(1.f, 1.f, 1.f, 1.f);
  const int h0 = blockIdx.y * a.hpg;
  const int h1 = min(h0 + a.hpg, a.H + a.Hkv);
  auto side = [&](const void* src, int64_t stride, void* dst, int64_t out_stride, const void* w,
                  int from, int to) {
    float4 w0 = one, w1 = one;
    if (w) {
      w0 = load_row4<T, VEC>(static_cast<const T*>(w) + lo);
      w1 = load_row4<T, VEC>(static_cast<const T*>(w) + hi);
    }
    norm_heads<T, D, VEC>(static_cast<const T*>(src) + tok * stride,
                          static_cast<T*>(dst) + tok * out_stride, from, to, w0, w1, c0, c1, s0,
                          s1, a.eps, lo, hi, live);
  };
  if (h0 < a.H) side(a.q, a.q_stride, a.q_out, a.qo_stride, a.w_q, h0, min(h1, a.H));
  if (h1 > a.H)
    side(a.k, a.k_stride, a.k_out, a.ko_stride, a.w_k, max(h0, a.H) - a.H, h1 - a.H);
}

template <typename T, int D>
int launch_norm_t(const NormRopeArgs& a, int vec, int sms, cudaStream_t s) {
  constexpr int kTok = kNormThreads / (D / 8);  // tokens per CTA
  const int64_t gx = (a.n + kTok - 1) / kTok;
  const int heads = a.H + a.Hkv;
  // pieces of heads: whole tokens where these fill the GPU (cos, sin and the
  // weights are read once), else one batch, which is what runs side by side (64
  // rows of 28 + 4 heads: 8 CTAs a token group, 2.4 us)
  NormRopeArgs b = a;
  b.hpg = gx >= 2 * sms ? heads : kBatch;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(gx),
                     static_cast<unsigned>((heads + b.hpg - 1) / b.hpg));
  cfg.blockDim = dim3(kNormThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(
      &cfg, vec ? qk_norm_rope_kernel<T, D, true> : qk_norm_rope_kernel<T, D, false>, b));
}

template <typename T>
int launch_norm_d(const NormRopeArgs& a, int vec, int sms, cudaStream_t s) {
  return a.D == 128 ? launch_norm_t<T, 128>(a, vec, sms, s) : launch_norm_t<T, 64>(a, vec, sms, s);
}

}  // namespace

int launch_qk_norm_rope(const NormRopeArgs& a, int dtype, int vec, int sms, cudaStream_t s) {
  switch (dtype) {
    case IR_DTYPE_F32: return launch_norm_d<float>(a, vec, sms, s);
    case IR_DTYPE_BF16: return launch_norm_d<__nv_bfloat16>(a, vec, sms, s);
    default: return launch_norm_d<__half>(a, vec, sms, s);
  }
}

}  // namespace irb
