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

// A group of D / 8 lanes takes heads [y * hpg, y * hpg + hpg) of one token;
// heads 0 .. H-1 are the query's, the rest the key's.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kNormThreads) qk_norm_rope_kernel(const NormRopeArgs a) {
  constexpr int LPR = D / 8;
  const int lane = threadIdx.x % LPR;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kNormThreads / LPR) + threadIdx.x / LPR;
  const bool live = t < a.n;
  const int64_t tok = live ? t : a.n - 1;  // idle groups follow along for the shuffles
  const int lo = lane * 4, hi = D / 2 + lane * 4;
  const float* cr = a.cos + tok * a.rope_stride;
  const float* sr = a.sin + tok * a.rope_stride;
  const float4 c0 = load_row4<float, VEC>(cr + lo), c1 = load_row4<float, VEC>(cr + hi);
  const float4 s0 = load_row4<float, VEC>(sr + lo), s1 = load_row4<float, VEC>(sr + hi);
  const float4 one = make_float4(1.f, 1.f, 1.f, 1.f);
  const T* wq = static_cast<const T*>(a.w_q);
  const T* wk = static_cast<const T*>(a.w_k);
  const int h0 = blockIdx.y * a.hpg;
  const int h1 = min(h0 + a.hpg, a.H + a.Hkv);
  float4 w0 = one, w1 = one;
  bool key = false;
  if (wq) w0 = load_row4<T, VEC>(wq + lo), w1 = load_row4<T, VEC>(wq + hi);
  for (int h = h0; h < h1; ++h) {
    if (h >= a.H && !key) {
      key = true;
      w0 = w1 = one;
      if (wk) w0 = load_row4<T, VEC>(wk + lo), w1 = load_row4<T, VEC>(wk + hi);
    }
    const T* src = h < a.H ? static_cast<const T*>(a.q) + tok * a.q_stride + h * D
                           : static_cast<const T*>(a.k) + tok * a.k_stride + (h - a.H) * D;
    const float4 x = load_row4<T, VEC>(src + lo), y = load_row4<T, VEC>(src + hi);
    float ss = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w + y.x * y.x + y.y * y.y +
               y.z * y.z + y.w * y.w;
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(ss * (1.f / D) + a.eps);
    const float4 u = make_float4(x.x * r * w0.x, x.y * r * w0.y, x.z * r * w0.z, x.w * r * w0.w);
    const float4 v = make_float4(y.x * r * w1.x, y.y * r * w1.y, y.z * r * w1.z, y.w * r * w1.w);
    if (live) {
      T* dst = h < a.H ? static_cast<T*>(a.q_out) + tok * a.qo_stride + h * D
                       : static_cast<T*>(a.k_out) + tok * a.ko_stride + (h - a.H) * D;
      store_row4<T, VEC>(dst + lo,
                         make_float4(u.x * c0.x - v.x * s0.x, u.y * c0.y - v.y * s0.y,
                                     u.z * c0.z - v.z * s0.z, u.w * c0.w - v.w * s0.w));
      store_row4<T, VEC>(dst + hi,
                         make_float4(v.x * c1.x + u.x * s1.x, v.y * c1.y + u.y * s1.y,
                                     v.z * c1.z + u.z * s1.z, v.w * c1.w + u.w * s1.w));
    }
  }
}

template <typename T, int D>
int launch_norm_t(const NormRopeArgs& a, int vec, int sms, cudaStream_t s) {
  constexpr int kTok = kNormThreads / (D / 8);  // tokens per CTA
  const int64_t gx = (a.n + kTok - 1) / kTok;
  const int heads = a.H + a.Hkv;
  NormRopeArgs b = a;
  b.hpg = heads;
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>((heads + b.hpg - 1) / b.hpg));
  if (vec)
    qk_norm_rope_kernel<T, D, true><<<grid, kNormThreads, 0, s>>>(b);
  else
    qk_norm_rope_kernel<T, D, false><<<grid, kNormThreads, 0, s>>>(b);
  return static_cast<int>(cudaGetLastError());
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
