// Causal attention of packed query rows over an 8-bit pool in fp32 on the CUDA
// cores: for q of 32 bits, for 16-bit calls that the tensor-core path cannot
// take (rows that are not 16-byte aligned, or asked for), and beside it for
// fp16 rows that attend values beyond fp16 (PrefillArgs::exact_from).
//
// A CTA takes 64 rows of one kv head, a row being a (query token, head of the
// group) pair, and walks the sequence's keys 64 at a time: the codes of a tile
// come through the block table 16 bytes a thread (the next tile's while the
// current one is computed), become fp32 rows in shared memory with their
// block's scale, and each of 256 threads computes 4 x 4 scores and 4 x D / 16
// outputs from registers, with an online softmax whose statistics live in the
// 16 lanes that share a row. Bound by FMA issue: 8 FMAs per 16-byte
// shared-memory read. 6 sequences of up to 300 rows over 700 more keys, 12 heads
// of 128, fp32: 283 us a call (5.8 GFLOP), where decoding every row takes 1500.
#include "kernels.h"
#include "quant.cuh"

namespace irb {

namespace {

constexpr int kM = 64;   // rows of a CTA
constexpr int kN = 64;   // keys of a tile
constexpr int kT = 256;  // threads: 16 row groups x 16 column groups
constexpr unsigned kAll32 = 0xffffffffu;

template <int D>
struct SmemQ8P {
  static constexpr int kKs = D + 4;   // padded: a phase's 8 rows hit distinct banks
  static constexpr int kPs = kN + 4;
  float q[kM][D];
  float k[kN][kKs];  // then the tile's weights, [kM][kPs]
  float v[kN][D];
  static_assert(kM * kPs <= kN * kKs, "the weights take the place of K");
  __device__ float* p(int r) { return &k[0][0] + r * kPs; }
};

// Tile `index` of the packed rows: its sequence and the tile within it, by the
// calling warp (sequences in order, ceil(rows / kM) tiles each).
__device__ __forceinline__ bool find_tile(const int32_t* q_start, int S, int total_q, int n_rep,
                                          int index, int* seq, int* tile, int* tiles) {
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  for (int base = 0; base < S; base += 32) {
    const int s = base + lane;
    int64_t t = 0;
    if (s < S) {
      const int64_t rows = static_cast<int64_t>(min(q_start[s + 1], total_q)) - q_start[s];
      t = rows > 0 && q_start[s] >= 0 ? (rows * n_rep + kM - 1) / kM : 0;
    }
    int64_t incl = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(kAll32, incl, o);
      if (lane >= o) incl += y;
    }
    const unsigned hit = __ballot_sync(kAll32, index < before + incl);
    if (hit) {
      const int l = __ffs(hit) - 1;
      const int64_t end = before + __shfl_sync(kAll32, incl, l);
      const int64_t n = __shfl_sync(kAll32, t, l);
      *seq = base + l;
      *tile = static_cast<int>(index - (end - n));
      *tiles = static_cast<int>(n);
      return true;
    }
    before += __shfl_sync(kAll32, incl, 31);
  }
  return false;
}

template <typename T, typename C, int D>
__global__ void __launch_bounds__(kT, 2)
    prefill_q8_kernel(const PrefillArgs a, const uint8_t* kp, const uint8_t* vp, const float* ks,
                      const float* vs) {
  extern __shared__ __align__(16) uint8_t raw[];
  SmemQ8P<D>& sm = *reinterpret_cast<SmemQ8P<D>*>(raw);
  __shared__ int s_seq, s_tile, s_tiles, s_nan;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int kvh = blockIdx.y;
  if (a.exact_from != nullptr && a.exact_from[a.S] == INT32_MAX) return;  // mostly
  if (tid < 32) {
    int seq = -1, tile = 0, tiles = 0;
    if (!find_tile(a.q_start, a.S, a.total_q, a.n_rep, blockIdx.x, &seq, &tile, &tiles)) seq = -1;
    if (tid == 0) s_seq = seq, s_tile = tile, s_tiles = tiles;
  }
  __syncthreads();
  if (s_seq < 0) return;
  const int sq = s_seq;
  // the last tiles of a sequence have the most keys: first
  const int tile = s_tiles - 1 - s_tile;
  const int q0 = a.q_start[sq];
  const int q_len = a.q_start[sq + 1] - q0, ctx = a.context_lens[sq];
  if (ctx < q_len || ctx > a.max_ctx || q0 + static_cast<int64_t>(q_len) > a.total_q) {
    if (tid == 0) set_err(a.err, IR_DEVERR_CONTEXT_LEN);
    return;
  }
  const int64_t m0 = static_cast<int64_t>(tile) * kM;
  const int64_t rows = static_cast<int64_t>(q_len) * a.n_rep;
  const int from = a.exact_from != nullptr ? a.exact_from[sq] : 0;  // first position to compute
  const int64_t last = (m0 + kM < rows ? m0 + kM : rows) - 1;
  const int keys = ctx - q_len + static_cast<int>(last / a.n_rep) + 1;  // the tile's last row's
  if (keys <= from) return;
  // this thread's rows: their position (-1: no row), and in the group
  int pos[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty * 4 + i;
    pos[i] = m < rows ? ctx - q_len + static_cast<int>(m / a.n_rep) : -1;
    if (pos[i] < from) pos[i] = -1;
  }

  // q rows, scaled so that scores come in log2 units
  for (int i = tid; i < kM * D; i += kT) {
    const int r = i / D, d = i % D;
    const int64_t m = m0 + r;
    float x = 0.f;
    if (m < rows) {
      const int64_t t = q0 + m / a.n_rep;
      const int h = kvh * a.n_rep + static_cast<int>(m % a.n_rep);
      x = DT<T>::to_f(static_cast<const T*>(a.q)[t * a.q_stride + static_cast<int64_t>(h) * D + d]);
    }
    sm.q[r][d] = x * a.scale_log2;
  }

  // a thread's 16-code chunks of a tile side, as loaded, with their scales
  constexpr int CPR = D / 16;             // chunks per row
  constexpr int CPT = kN * CPR / kT;      // chunks per thread and side
  uint4 kc[CPT], vc[CPT];
  float ksc[CPT], vsc[CPT];
  const int32_t* btr = a.block_tables + sq * a.bt_stride;
  auto load = [&](int k0) {
#pragma unroll
    for (int u = 0; u < CPT; ++u) {
      const int i = tid + u * kT, key = k0 + i / CPR, c = i % CPR;
      kc[u] = vc[u] = make_uint4(0u, 0u, 0u, 0u);
      ksc[u] = vsc[u] = 0.f;
      if (key >= keys) continue;
      const int64_t id = btr[key / a.bs];
      if (id < 0 || id >= a.num_blocks) {
        if (c == 0) set_err(a.err, IR_DEVERR_BLOCK_ID);
        continue;
      }
      const int64_t at = ((id * a.bs + key % a.bs) * a.Hkv + kvh) * D + c * 16;
      kc[u] = *reinterpret_cast<const uint4*>(kp + at);
      vc[u] = *reinterpret_cast<const uint4*>(vp + at);
      ksc[u] = ks[id * a.Hkv + kvh];
      vsc[u] = vs[id * a.Hkv + kvh];
    }
  };
  auto store = [&]() {
    bool nan = false;
#pragma unroll
    for (int u = 0; u < CPT; ++u) {
      const int i = tid + u * kT, r = i / CPR, c = (i % CPR) * 16;
      const uint32_t kw[4] = {kc[u].x, kc[u].y, kc[u].z, kc[u].w};
      const uint32_t vw[4] = {vc[u].x, vc[u].y, vc[u].z, vc[u].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float4 x = decode4<C>(kw[e]), y = decode4<C>(vw[e]);
        const float4 z = make_float4(y.x * vsc[u], y.y * vsc[u], y.z * vsc[u], y.w * vsc[u]);
        *reinterpret_cast<float4*>(&sm.k[r][c + 4 * e]) =
            make_float4(x.x * ksc[u], x.y * ksc[u], x.z * ksc[u], x.w * ksc[u]);
        *reinterpret_cast<float4*>(&sm.v[r][c + 4 * e]) = z;
        // 0 * z is not 0: a row must not see it before its position
        const float t = (z.x + z.y + z.z + z.w) * 0.f;
        nan = nan || t != 0.f;
      }
    }
    if (nan) s_nan = 1;
  };

  constexpr int CO = D / 16;  // output columns of a thread: 4 at 64 h + 4 tx
  float o[4][CO], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < CO; ++c) o[i][c] = 0.f;
  }
  load(0);
  for (int k0 = 0; k0 < keys; k0 += kN) {
    __syncthreads();  // the tile before is read (and q is written)
    if (tid == 0) s_nan = 0;
    __syncthreads();
    store();
    __syncthreads();
    if (k0 + kN < keys) load(k0 + kN);
    const bool careful = s_nan != 0;

    float s[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      float4 x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(&sm.q[ty * 4 + i][d]);
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(&sm.k[tx + 16 * j][d]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[i][j] = fmaf(x[i].x, y[j].x, s[i][j]);
          s[i][j] = fmaf(x[i].y, y[j].y, s[i][j]);
          s[i][j] = fmaf(x[i].z, y[j].z, s[i][j]);
          s[i][j] = fmaf(x[i].w, y[j].w, s[i][j]);
        }
    }
    __syncthreads();  // K is read: the weights take its place
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (k0 + tx + 16 * j > pos[i]) s[i][j] = -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kAll32, mx, w));
      const float top = fmaxf(m[i], mx);
      const float use = top == -INFINITY ? 0.f : top;
      const float alpha = ex2(m[i] - use);
      m[i] = top;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = ex2(s[i][j] - use);
        sum += p;
        sm.p(ty * 4 + i)[tx + 16 * j] = p;
      }
      l[i] = l[i] * alpha + sum;  // (this lane's columns; added up at the end)
#pragma unroll
      for (int c = 0; c < CO; ++c) o[i][c] *= alpha;
    }
    __syncwarp();  // a row's 16 lanes are in one warp
    if (!careful) {
#pragma unroll 2
      for (int k = 0; k < kN; k += 4) {
        float4 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const float4*>(sm.p(ty * 4 + i) + k);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
          for (int h = 0; h < CO / 4; ++h) {
            const float4 y = *reinterpret_cast<const float4*>(&sm.v[k + kk][64 * h + tx * 4]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float w = kk == 0 ? p[i].x : kk == 1 ? p[i].y : kk == 2 ? p[i].z : p[i].w;
              o[i][4 * h] = fmaf(w, y.x, o[i][4 * h]);
              o[i][4 * h + 1] = fmaf(w, y.y, o[i][4 * h + 1]);
              o[i][4 * h + 2] = fmaf(w, y.z, o[i][4 * h + 2]);
              o[i][4 * h + 3] = fmaf(w, y.w, o[i][4 * h + 3]);
            }
          }
      }
    } else {
      for (int k = 0; k < kN; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (k0 + k > pos[i]) continue;
          const float w = sm.p(ty * 4 + i)[k];
#pragma unroll
          for (int c = 0; c < CO; ++c)
            o[i][c] = fmaf(w, sm.v[k][64 * (c / 4) + tx * 4 + c % 4], o[i][c]);
        }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) l[i] += __shfl_xor_sync(kAll32, l[i], w);
    if (pos[i] < 0) continue;
    const int64_t mr = m0 + ty * 4 + i;
    const int64_t t = q0 + mr / a.n_rep;
    const int h = kvh * a.n_rep + static_cast<int>(mr % a.n_rep);
    const float f = l[i] == 0.f ? 0.f : 1.f / l[i];
    T* dst = static_cast<T*>(a.out) + t * a.out_stride + static_cast<int64_t>(h) * D;
#pragma unroll
    for (int c = 0; c < CO; ++c) dst[64 * (c / 4) + tx * 4 + c % 4] = DT<T>::from_f(o[i][c] * f);
  }
}

template <typename T, typename C, int D>
int launch_p(const PrefillArgs& a, const void* kp, const void* vp, const float* ks,
             const float* vs, cudaStream_t s) {
  auto kern = prefill_q8_kernel<T, C, D>;
  constexpr int bytes = static_cast<int>(sizeof(SmemQ8P<D>));
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return static_cast<int>(e);
  // at most this many tiles: every sequence's last one may be short
  const int64_t tiles = (static_cast<int64_t>(a.total_q) * a.n_rep + kM - 1) / kM + a.S;
  if (tiles > INT32_MAX) return static_cast<int>(cudaErrorInvalidConfiguration);
  kern<<<dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(a.Hkv)), kT, bytes, s>>>(
      a, static_cast<const uint8_t*>(kp), static_cast<const uint8_t*>(vp), ks, vs);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, typename C>
int by_d(const PrefillArgs& a, const void* kp, const void* vp, const float* ks, const float* vs,
         cudaStream_t s) {
  return a.D == 128 ? launch_p<T, C, 128>(a, kp, vp, ks, vs, s)
                    : launch_p<T, C, 64>(a, kp, vp, ks, vs, s);
}

template <typename T>
int by_c(int fmt, const PrefillArgs& a, const void* kp, const void* vp, const float* ks,
         const float* vs, cudaStream_t s) {
  return fmt == IR_KV_INT8 ? by_d<T, int8_t>(a, kp, vp, ks, vs, s)
                           : by_d<T, e4m3_t>(a, kp, vp, ks, vs, s);
}

}  // namespace

int launch_prefill_q8(const PrefillArgs& a, const void* k_pool, const void* v_pool,
                      const float* k_scale, const float* v_scale, int dtype, int fmt,
                      cudaStream_t s) {
  auto run = [&](auto by) {
    return by(fmt, a, k_pool, v_pool, k_scale, v_scale, s);
  };
  switch (dtype) {
    case IR_DTYPE_F32: return run(by_c<float>);
    case IR_DTYPE_BF16: return run(by_c<__nv_bfloat16>);
    default: return run(by_c<__half>);
  }
}

}  // namespace irb
