// The 8-bit K/V cache: quantising write, gather, and whole blocks read back as
// rows of the compute type (the pool a prefill call attends over).
//
// The write. Every (block, kv head) of a pool has one scale, so the rows a
// call brings to one block are handled together, by one CTA, whatever order
// they come in: the call's tokens are grouped by block, the group's first
// finder owns the block, and src[offset] holds the token that brings that
// row (the last one where a slot appears twice). A warp takes one (K or V,
// kv head) of the block: it finds the largest magnitude of the new rows,
//   s' = max(s, scale_for(amax))          (s counts as 0 when row 0 is new),
// rescales the codes that stay if s' > s, and writes the new codes. Nothing
// is summed, so the result does not depend on the order of the tokens.
#include "kernels.h"
#include "quant.cuh"

namespace irb {

namespace {

constexpr int kQThreads = 256;
constexpr int kQWarps = kQThreads / 32;
constexpr unsigned kAll = 0xffffffffu;

struct Q8WriteArgs {
  const void* src[2];  // k, v rows
  int64_t stride[2];   // elements between tokens
  uint8_t* pool[2];
  float* scale[2];  // [num_blocks, Hkv]
  const int64_t* slots;
  int64_t n, num_slots;
  int Hkv, D, bs;
  int vec;  // rows are read in 4-element vectors
  int32_t* err;
};

// Four elements of a row as fp32.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p, int vec) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      return *reinterpret_cast<const float4*>(p);
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(p);
      const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
      return make_float4(a.x, a.y, b.x, b.y);
    }
  }
  return make_float4(DT<T>::to_f(p[0]), DT<T>::to_f(p[1]), DT<T>::to_f(p[2]), DT<T>::to_f(p[3]));
}

__device__ __forceinline__ bool finite(float x) {
  return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
}

// One (side, kv head) of block `blk`, by one warp; src[] in shared memory.
// Lanes cover D in groups of 4 elements, RP = 128 / D rows at a time.
template <typename T, typename C>
__device__ void quantise_task(const Q8WriteArgs& a, int64_t blk, const int* src, int side, int h) {
  constexpr bool kInt = std::is_same<C, int8_t>::value;
  const int lane = threadIdx.x & 31;
  const int lpr = a.D / 4;         // lanes per row
  const int rp = 32 / lpr;         // rows per pass
  const int sub = lane / lpr, col = (lane % lpr) * 4;
  const T* in = reinterpret_cast<const T*>(a.src[side]) + static_cast<int64_t>(h) * a.D + col;
  const int64_t stride = a.stride[side];
  const int64_t row_bytes = static_cast<int64_t>(a.Hkv) * a.D;
  uint8_t* dst = a.pool[side] + (blk * a.bs) * row_bytes + static_cast<int64_t>(h) * a.D + col;

  float amax = 0.f;
  bool bad = false;
#pragma unroll 4
  for (int r = sub; r < a.bs; r += rp) {
    const int t = src[r];
    if (t < 0) continue;
    const float4 x = load4<T>(in + t * stride, a.vec);
    const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (finite(v[i])) amax = fmaxf(amax, fabsf(v[i]));
      else bad = true;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(kAll, amax, o));
  bad = __any_sync(kAll, bad);

  float* sp = a.scale[side] + blk * a.Hkv + h;
  const bool begun = src[0] >= 0;
  const float old = begun ? 0.f : *sp;
  const float need = scale_for<C>(amax);
  float now = old > need ? old : need;
  // int8 has no code for a value that is not finite: its block reads as NaN
  // until it is begun again
  if (kInt && (bad || old != old)) now = __uint_as_float(0x7fc00000u);
  __syncwarp();  // every lane has read the old scale
  if (lane == 0) *sp = now;

  if (!begun && now != old && now == now) {
    // rescale the codes that stay
    const float inv = pow2_reciprocal(now);
    const float ratio = inv != 0.f ? old * inv : old / now;
    for (int r = sub; r < a.bs; r += rp) {
      if (src[r] >= 0) continue;
      uint32_t* p = reinterpret_cast<uint32_t*>(dst + r * row_bytes);
      float4 x = decode4<C>(*p);
      x.x *= ratio;
      x.y *= ratio;
      x.z *= ratio;
      x.w *= ratio;
      *p = encode4<C>(x);
    }
  }
  const float inv = pow2_reciprocal(now);
#pragma unroll 4
  for (int r = sub; r < a.bs; r += rp) {
    const int t = src[r];
    if (t < 0) continue;
    float4 x = load4<T>(in + t * stride, a.vec);
    float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!finite(v[i])) v[i] = __uint_as_float(0x7fc00000u);
      else v[i] = inv != 0.f ? v[i] * inv : v[i] / now;
    }
    *reinterpret_cast<uint32_t*>(dst + r * row_bytes) =
        encode4<C>(make_float4(v[0], v[1], v[2], v[3]));
  }
}

// One CTA per token (x) and group of kQWarps tasks (y): the CTA of a block's
// first token owns the block; it finds the others by reading all slots, which
// takes no launch and no scratch of its own (for calls of few tokens).
template <typename T, typename C>
__global__ void __launch_bounds__(kQThreads) write_scan_kernel(const Q8WriteArgs a) {
  extern __shared__ int src[];
  const int64_t i = blockIdx.x;
  const int64_t s = a.slots[i];
  if (s < 0) return;  // padding row
  if (s >= a.num_slots) {
    if (threadIdx.x == 0 && blockIdx.y == 0) set_err(a.err, IR_DEVERR_SLOT);
    return;
  }
  const int64_t blk = s / a.bs, lo = blk * a.bs;
  for (int r = threadIdx.x; r < a.bs; r += kQThreads) src[r] = -1;
  __syncthreads();
  bool earlier = false;
  for (int64_t j = threadIdx.x; j < a.n; j += kQThreads) {
    const int64_t off = a.slots[j] - lo;
    if (off < 0 || off >= a.bs) continue;
    earlier = earlier || j < i;
    atomicMax(&src[off], static_cast<int>(j));
  }
  if (__syncthreads_or(earlier)) return;
  const int task = blockIdx.y * kQWarps + (threadIdx.x >> 5);
  if (task < 2 * a.Hkv) quantise_task<T, C>(a, blk, src, task / a.Hkv, task % a.Hkv);
}

// Larger calls: the tokens' runs (neighbours in one block) are linked per
// block first. head[blk] is the block's last linked run + 1 (0: none), next[i]
// the run before it, owners[] the blocks in the order they were found.
struct Q8Links {
  int* count;
  int* head;
  int* next;
  int* owners;
};

__global__ void link_runs_kernel(const int64_t* slots, int64_t n, int64_t num_slots, int bs,
                                 const Q8Links l, int32_t* err) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t s = slots[i];
  if (s < 0) return;
  if (s >= num_slots) {
    set_err(err, IR_DEVERR_SLOT);
    return;
  }
  const int64_t blk = s / bs;
  if (i > 0) {
    const int64_t off = slots[i - 1] - blk * bs;
    if (off >= 0 && off < bs) return;  // not the first of its run
  }
  const int prev = atomicExch(&l.head[blk], static_cast<int>(i) + 1);
  l.next[i] = prev;
  if (prev == 0) l.owners[atomicAdd(l.count, 1)] = static_cast<int>(blk);
}

template <typename T, typename C>
__global__ void __launch_bounds__(kQThreads) write_runs_kernel(const Q8WriteArgs a,
                                                               const Q8Links l) {
  extern __shared__ int src[];
  const int count = *l.count;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int o = blockIdx.x; o < count; o += gridDim.x) {
    const int64_t blk = l.owners[o], lo = blk * a.bs;
    for (int r = threadIdx.x; r < a.bs; r += kQThreads) src[r] = -1;
    __syncthreads();
    if (warp == 0) {
      for (int run = l.head[blk]; run != 0;) {
        const int64_t first = run - 1;
        for (int64_t j = first + lane;; j += 32) {
          const int64_t off = j < a.n ? a.slots[j] - lo : -1;
          const bool in = off >= 0 && off < a.bs;
          // a run ends at its first token of another block
          const unsigned m = __ballot_sync(kAll, in);
          const int len = m == kAll ? 32 : __ffs(~m) - 1;
          if (lane < len) atomicMax(&src[off], static_cast<int>(j));
          if (len < 32) break;
        }
        run = l.next[first];
      }
    }
    __syncthreads();
    for (int task = warp; task < 2 * a.Hkv; task += kQWarps)
      quantise_task<T, C>(a, blk, src, task / a.Hkv, task % a.Hkv);
    __syncthreads();
  }
}

// 16 codes to 16 values of T, multiplied by the scale in fp32 and rounded once;
// finite values beyond T's range saturate.
template <typename T>
__device__ __forceinline__ float saturate(float x) {
  if constexpr (std::is_same<T, __half>::value) {
    if (fabsf(x) > 65504.f && finite(x)) return copysignf(65504.f, x);
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const float top = __uint_as_float(0x7f7f0000u);
    if (fabsf(x) > top && finite(x)) return copysignf(top, x);
  }
  return x;
}

template <typename T, typename C>
__device__ __forceinline__ void store16(T* out, uint4 codes, float s, int vec) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 x = decode4<C>(w[i]);
    const float a = saturate<T>(x.x * s), b = saturate<T>(x.y * s), c = saturate<T>(x.z * s),
                d = saturate<T>(x.w * s);
    T* p = out + 4 * i;
    if (!vec) {
      p[0] = DT<T>::from_f(a);
      p[1] = DT<T>::from_f(b);
      p[2] = DT<T>::from_f(c);
      p[3] = DT<T>::from_f(d);
    } else if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
    } else {
      *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(a, b), pack2<T>(c, d));
    }
  }
}

template <typename T, typename C>
__global__ void gather_q8_kernel(T* out, const uint8_t* pool, const float* scale,
                                 const int64_t* slots, int64_t n, int Hkv, int D, int bs,
                                 int64_t num_slots, int vec, int32_t* err) {
  const int cpr = Hkv * D / 16;  // 16-code chunks per row
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= n * cpr) return;
  const int64_t r = i / cpr;
  const int c = static_cast<int>(i - r * cpr);
  const int64_t s = slots[r];
  T* dst = out + i * 16;
  if (s < 0 || s >= num_slots) {
    if (c == 0) set_err(err, IR_DEVERR_SLOT);
    store16<T, C>(dst, make_uint4(0, 0, 0, 0), 0.f, vec);
    return;
  }
  const uint4 codes = *reinterpret_cast<const uint4*>(pool + (s * cpr + c) * 16);
  store16<T, C>(dst, codes, scale[s / bs * Hkv + c * 16 / D], vec);
}

// Blocks of the sequences' histories, each to its own place in a pool of T.
template <typename T, typename C>
__global__ void expand_blocks_kernel(T* kout, T* vout, const uint8_t* kp, const uint8_t* vp,
                                     const float* ks, const float* vs, const int32_t* bt,
                                     int64_t bt_stride, const int32_t* ctx, int max_blocks,
                                     int64_t num_blocks, int Hkv, int D, int bs) {
  const int sq = blockIdx.x;
  const int64_t c0 = ctx[sq];
  const int cpr = Hkv * D / 16;
  const int64_t chunks = static_cast<int64_t>(bs) * cpr;
  for (int j = blockIdx.y; j < max_blocks && static_cast<int64_t>(j) * bs < c0; j += gridDim.y) {
    const int64_t id = bt[sq * bt_stride + j];
    if (id < 0 || id >= num_blocks) continue;  // the attention kernel reports it
    const int64_t base = id * chunks;
    for (int64_t i = threadIdx.x; i < chunks; i += blockDim.x) {
      const int h = static_cast<int>(i % cpr) * 16 / D;
      const uint4 kc = reinterpret_cast<const uint4*>(kp)[base + i];
      const uint4 vc = reinterpret_cast<const uint4*>(vp)[base + i];
      store16<T, C>(kout + (base + i) * 16, kc, ks[id * Hkv + h], 1);
      store16<T, C>(vout + (base + i) * 16, vc, vs[id * Hkv + h], 1);
    }
  }
}

template <typename F>
int by_format(int fmt, F f) {
  return fmt == IR_KV_INT8 ? f(int8_t{}) : f(e4m3_t{});
}
template <typename F>
int by_type(int dtype, F f) {
  switch (dtype) {
    case IR_DTYPE_F32: return f(float{});
    case IR_DTYPE_BF16: return f(__nv_bfloat16{});
    default: return f(__half{});
  }
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Calls of up to this many tokens find each block's rows by reading all slots.
constexpr int64_t kScanTokens = 1024;

}  // namespace

size_t cache_write_q8_workspace(int64_t n, int64_t num_blocks) {
  if (n <= kScanTokens) return 0;
  const int64_t owners = n < num_blocks ? n : num_blocks;
  return align256(static_cast<size_t>(num_blocks + 1) * 4) + align256(static_cast<size_t>(n) * 4) +
         align256(static_cast<size_t>(owners) * 4);
}

int launch_cache_write_q8(const void* k, const void* v, int64_t k_stride, int64_t v_stride,
                          void* k_pool, void* v_pool, float* k_scale, float* v_scale,
                          const int64_t* slots, int64_t n, int Hkv, int D, int bs,
                          int64_t num_slots, int dtype, int fmt, void* ws, int sms, int32_t* err,
                          cudaStream_t stream) {
  const int eb = dtype == IR_DTYPE_F32 ? 4 : 2;
  Q8WriteArgs a{};
  a.src[0] = k;
  a.src[1] = v;
  a.stride[0] = k_stride;
  a.stride[1] = v_stride;
  a.pool[0] = static_cast<uint8_t*>(k_pool);
  a.pool[1] = static_cast<uint8_t*>(v_pool);
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.slots = slots;
  a.n = n;
  a.num_slots = num_slots;
  a.Hkv = Hkv;
  a.D = D;
  a.bs = bs;
  a.vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % (4 * eb)) == 0 &&
          k_stride % 4 == 0 && v_stride % 4 == 0;
  a.err = err;
  const size_t smem = static_cast<size_t>(bs) * 4;
  if (n <= kScanTokens) {
    const dim3 grid(static_cast<unsigned>(n), (2 * Hkv + kQWarps - 1) / kQWarps);
    return by_type(dtype, [&](auto t) {
      return by_format(fmt, [&](auto c) {
        write_scan_kernel<decltype(t), decltype(c)><<<grid, kQThreads, smem, stream>>>(a);
        return static_cast<int>(cudaGetLastError());
      });
    });
  }
  const int64_t num_blocks = num_slots / bs;
  uint8_t* w = static_cast<uint8_t*>(ws);
  const size_t heads = align256(static_cast<size_t>(num_blocks + 1) * 4);
  Q8Links l;
  l.count = reinterpret_cast<int*>(w);
  l.head = l.count + 1;
  l.next = reinterpret_cast<int*>(w + heads);
  l.owners = reinterpret_cast<int*>(w + heads + align256(static_cast<size_t>(n) * 4));
  cudaError_t e = cudaMemsetAsync(w, 0, heads, stream);
  if (e != cudaSuccess) return static_cast<int>(e);
  link_runs_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, stream>>>(
      slots, n, num_slots, bs, l, err);
  e = cudaGetLastError();
  if (e != cudaSuccess) return static_cast<int>(e);
  int64_t grid = n < num_blocks ? n : num_blocks;
  if (grid > static_cast<int64_t>(sms) * 8) grid = static_cast<int64_t>(sms) * 8;
  return by_type(dtype, [&](auto t) {
    return by_format(fmt, [&](auto c) {
      write_runs_kernel<decltype(t), decltype(c)>
          <<<static_cast<unsigned>(grid), kQThreads, smem, stream>>>(a, l);
      return static_cast<int>(cudaGetLastError());
    });
  });
}

int launch_cache_gather_q8(void* out, const void* pool, const float* scale, const int64_t* slots,
                           int64_t n, int Hkv, int D, int bs, int64_t num_slots, int dtype,
                           int fmt, int32_t* err, cudaStream_t stream) {
  const int64_t work = n * (static_cast<int64_t>(Hkv) * D / 16);
  const unsigned grid = static_cast<unsigned>((work + 255) / 256);
  const int vec = reinterpret_cast<uintptr_t>(out) % 16 == 0;
  return by_type(dtype, [&](auto t) {
    return by_format(fmt, [&](auto c) {
      using T = decltype(t);
      gather_q8_kernel<T, decltype(c)><<<grid, 256, 0, stream>>>(
          static_cast<T*>(out), static_cast<const uint8_t*>(pool), scale, slots, n, Hkv, D, bs,
          num_slots, vec, err);
      return static_cast<int>(cudaGetLastError());
    });
  });
}

int launch_expand_blocks(void* k_out, void* v_out, const void* k_pool, const void* v_pool,
                         const float* k_scale, const float* v_scale, const int32_t* bt,
                         int64_t bt_stride, const int32_t* ctx, int S, int max_blocks,
                         int64_t num_blocks, int Hkv, int D, int bs, int dtype, int fmt,
                         cudaStream_t stream) {
  if (S == 0 || max_blocks == 0) return 0;
  const dim3 grid(static_cast<unsigned>(S),
                  static_cast<unsigned>(max_blocks < 4096 ? max_blocks : 4096));
  return by_type(dtype, [&](auto t) {
    return by_format(fmt, [&](auto c) {
      using T = decltype(t);
      expand_blocks_kernel<T, decltype(c)><<<grid, 256, 0, stream>>>(
          static_cast<T*>(k_out), static_cast<T*>(v_out), static_cast<const uint8_t*>(k_pool),
          static_cast<const uint8_t*>(v_pool), k_scale, v_scale, bt, bt_stride, ctx, max_blocks,
          num_blocks, Hkv, D, bs);
      return static_cast<int>(cudaGetLastError());
    });
  });
}

}  // namespace irb
