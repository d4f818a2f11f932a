// The 8-bit K/V cache: quantising write, gather, and whole blocks read back as
// rows of the compute type (the pool a prefill call attends over).
//
// The write. Every (block, kv head) of a pool has one scale, so the rows a
// call brings to one block are handled together, whatever order they come in:
// the call's tokens are grouped by block, and src(offset) is the token that
// brings that row (the last one where a slot appears twice). A warp takes one
// (K or V, kv head) of the block: it finds the largest magnitude of the new
// rows,
//   s' = max(s, scale_for(amax))          (s counts as 0 when row 0 is new),
// rescales the codes that stay if s' > s, and writes the new codes. Nothing
// is summed, so the result does not depend on the order of the tokens. Up to 2048
// elements of a block's rows a warp (16 rows of 128) wait in registers, or in
// shared memory where the next task's are copied meanwhile, between the maximum
// and the codes; rows of a larger block, or with a value that is not finite, are
// read again for the codes.
//
// Large calls wait for their reads: 32768 rows of 4 heads of 128, bf16, move 101 MB
// in 24.4 us (15.6 at the copy rate), 23 without the stores, HBM 39 % busy; 5-6 of
// them are the two small grids that group the rows. Blocks of more than 2048
// elements a head have no streamed form (8192 rows in blocks of 64: 13.4 us,
// 8.8 in blocks of 16). Small calls are one launch (64 rows 3.3 us, 777 int8 5.6).
#include "kernels.h"
#include "quant.cuh"

namespace irb {

namespace {

constexpr int kQThreads = 256;
constexpr int kQWarps = kQThreads / 32;
// Calls of up to this many tokens find each block's rows by reading all slots:
// one launch instead of three. 1024 rows of one prompt take 6.9 us so, 6.1 with
// linked runs, but each launch costs the host 2-3 us more; 1024 rows appended to
// as many blocks take 11.1 (the scan is quadratic, so not for much longer calls).
constexpr int64_t kScanTokens = 1024;
constexpr unsigned kAll = 0xffffffffu;

// The next grid of the stream may be set up now / wait for the one before.
__device__ __forceinline__ void let_next_grid_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void wait_prior_grid() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Launch with programmatic stream serialization: the grid may be set up while
// the one before it in the stream still runs, and waits for it itself.
template <typename... P, typename... A>
int launch_behind(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                  A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, P(args)...));
}

struct Q8WriteArgs {
  const void* src[2];  // k, v rows
  int stride[2];       // elements between tokens
  uint8_t* pool[2];
  float* scale[2];  // [num_blocks, Hkv]
  const int64_t* slots;
  int64_t n, num_slots;
  int Hkv, D, bs;
  int32_t* err;
};

__device__ __forceinline__ bool finite(float x) {
  return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
}

// Larger of two pairs; NaN where either is NaN.
template <typename T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value)
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Eight elements of a row, as loaded.
template <typename T> struct Eight {
  uint4 w;
  template <bool VEC>
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC) {
      w = *reinterpret_cast<const uint4*>(p);
    } else {
      const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
      uint32_t v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = u[2 * i] | (static_cast<uint32_t>(u[2 * i + 1]) << 16);
      w = make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
  // Running maximum of the magnitudes, two halves side by side; NaN stays.
  __device__ __forceinline__ uint32_t top(uint32_t m) const {
    return max2<T>(max2<T>(m, max2<T>(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu)),
                   max2<T>(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
  }
  static __device__ __forceinline__ float magnitude(uint32_t m) {
    return unpack2<T>(max2<T>(m, m >> 16)).x;
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(u[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
};
template <> struct Eight<float> {
  float4 a, b;
  template <bool VEC>
  __device__ __forceinline__ void load(const float* p) {
    if constexpr (VEC) {
      a = reinterpret_cast<const float4*>(p)[0];
      b = reinterpret_cast<const float4*>(p)[1];
    } else {
      a = make_float4(p[0], p[1], p[2], p[3]);
      b = make_float4(p[4], p[5], p[6], p[7]);
    }
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  // (the magnitudes' bits are in the order of the magnitudes, NaN above all)
  __device__ __forceinline__ uint32_t top(uint32_t m) const {
    float v[8];
    values(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
  }
  static __device__ __forceinline__ float magnitude(uint32_t m) { return __uint_as_float(m); }
};

template <typename C>
__device__ __forceinline__ uint2 encode8(const float (&v)[8]) {
  return make_uint2(encode4<C>(make_float4(v[0], v[1], v[2], v[3])),
                    encode4<C>(make_float4(v[4], v[5], v[6], v[7])));
}

// The scale of a (block, side, head) after the new rows (largest finite
// magnitude amax; `bad`: one was not finite), written by lane 0.
template <typename C>
__device__ __forceinline__ float settle_scale(float amax, bool bad, bool begun, float before,
                                              float* sp) {
  constexpr bool kInt = std::is_same<C, int8_t>::value;
  const float old = begun ? 0.f : before;
  const float need = scale_for<C>(amax);
  float now = old > need ? old : need;
  // int8 has no code for a value that is not finite: its block reads as NaN
  // until it is begun again
  if (kInt && (bad || old != old)) now = __uint_as_float(0x7fc00000u);
  if ((threadIdx.x & 31) == 0) *sp = now;
  return now;
}

// The codes that stay, moved from scale `old` to `now`.
template <typename C, typename Src>
__device__ __forceinline__ void rescale_rest(const Q8WriteArgs& a, Src src, uint8_t* dst,
                                             int row_bytes, int rp, int sub, float old,
                                             float now) {
  const float inv = pow2_reciprocal(now);
  const float ratio = inv != 0.f ? old * inv : old / now;
  for (int base = 0; base < a.bs; base += rp) {
    const int r = base + sub;
    const int t = src(r < a.bs ? r : 0);
    if (r >= a.bs || t >= 0) continue;
    uint2* p = reinterpret_cast<uint2*>(dst + r * row_bytes);
    const uint2 c = *p;
    const float4 f = decode4<C>(c.x), g = decode4<C>(c.y);
    const float v[8] = {f.x * ratio, f.y * ratio, f.z * ratio, f.w * ratio,
                        g.x * ratio, g.y * ratio, g.z * ratio, g.w * ratio};
    *p = encode8<C>(v);
  }
}

constexpr int kPass = 8;  // passes of rows that a warp holds at once

// Codes of the new rows held in x (bit u of have: pass u is one), all finite;
// `row` is this lane's place in pass 0, `apart` the bytes between passes.
template <typename T, typename C>
__device__ __forceinline__ void encode_rows(const Eight<T> (&x)[kPass], uint32_t have, float inv,
                                            uint8_t* row, int apart) {
#pragma unroll
  for (int u = 0; u < kPass; ++u) {
    float v[8];
    x[u].values(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= inv;
    const uint2 c = encode8<C>(v);
    if ((have >> u) & 1u) *reinterpret_cast<uint2*>(row + u * apart) = c;
  }
}

// One (side, kv head) of block `blk`, by one warp. Lanes cover D in groups of
// 8 elements, 256 / D rows at a time, kPass such passes at once. src(r) is
// called by all lanes of the warp together.
template <typename T, typename C, bool VEC, typename Src>
__device__ __forceinline__ void quantise_task(const Q8WriteArgs& a, int64_t blk, Src src, int side,
                                              int h) {
  const int lane = threadIdx.x & 31;
  const int sh = a.D == 128 ? 4 : 3;  // log2 of the lanes per row
  const int rp = 32 >> sh;            // rows per pass
  const int sub = lane >> sh, col = (lane & ((1 << sh) - 1)) * 8;
  const T* in = reinterpret_cast<const T*>(a.src[side]) + h * a.D + col;
  const int stride = a.stride[side];
  const int row_bytes = a.Hkv * a.D;  // (a block's bytes stay below 2^31)
  uint8_t* dst = a.pool[side] + blk * a.bs * row_bytes + (h * a.D + col);
  float* sp = a.scale[side] + blk * a.Hkv + h;
  const float before = *sp;  // (loaded beside the rows)
  const bool begun = src(0) >= 0;
  // the last of the block's new rows stands in for those that are not new,
  // which leaves the maximum as it is and the loads without a branch
  int some = -1;
  for (int base = 0; base < a.bs; base += 32)
    some = max(some, src(base + lane < a.bs ? base + lane : 0));
  some = __reduce_max_sync(kAll, some);

  Eight<T> x[kPass];
  uint32_t have = 0;  // bit u: pass u of the rows in registers is a new row
  auto load = [&](int base) {
    have = 0;
#pragma unroll
    for (int u = 0; u < kPass; ++u) {
      const int r = base + u * rp + sub;
      int t = src(r < a.bs ? r : 0);
      if (r < a.bs && t >= 0)
        have |= 1u << u;
      else
        t = some;
      x[u].template load<VEC>(in + static_cast<int64_t>(t) * stride);
    }
  };
  const int chunk = kPass * rp;
  uint32_t m = 0;
  for (int base = 0; base < a.bs; base += chunk) {
    load(base);
#pragma unroll
    for (int u = 0; u < kPass; ++u) m = x[u].top(m);
  }
  float amax = Eight<T>::magnitude(m);
  const bool bad = __any_sync(kAll, !finite(amax));
  if (bad) {  // the largest finite one
    amax = 0.f;
    for (int base = 0; base < a.bs; base += chunk) {
      load(base);
#pragma unroll
      for (int u = 0; u < kPass; ++u) {
        float v[8];
        x[u].values(v);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (finite(v[i])) amax = fmaxf(amax, fabsf(v[i]));
      }
    }
  }
  // (bits of magnitudes are in their order)
  amax = __uint_as_float(__reduce_max_sync(kAll, __float_as_uint(amax)));

  const float now = settle_scale<C>(amax, bad, begun, before, sp);
  const float inv = pow2_reciprocal(now);
  if (!begun && now != before && now == now)
    rescale_rest<C>(a, src, dst, row_bytes, rp, sub, before, now);
  if (!bad && inv != 0.f) {
    // every value finite and the scale a power of two: no case to tell apart
    for (int base = 0; base < a.bs; base += chunk) {
      if (chunk < a.bs) load(base);
      encode_rows<T, C>(x, have, inv, dst + (base + sub) * row_bytes, rp * row_bytes);
    }
    return;
  }
  const float nan = __uint_as_float(0x7fc00000u);
  for (int base = 0; base < a.bs; base += rp) {
    const int r = base + sub;
    const int t = src(r < a.bs ? r : 0);
    if (r >= a.bs || t < 0) continue;
    Eight<T> one;
    one.template load<VEC>(in + static_cast<int64_t>(t) * stride);
    float v[8];
    one.values(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = finite(v[i]) ? v[i] / now : nan;
    *reinterpret_cast<uint2*>(dst + r * row_bytes) = encode8<C>(v);
  }
}

// One CTA per token (x) and group of kQWarps tasks (y): the CTA of a block's
// first token owns the block; it finds the others by reading all slots, which
// takes no launch and no scratch of its own (for calls of few tokens).
template <typename T, typename C, bool VEC>
__global__ void __launch_bounds__(kQThreads) write_scan_kernel(const Q8WriteArgs a) {
  extern __shared__ int src[];
  wait_prior_grid();
  const int i = blockIdx.x;
  // every slot at once: one round trip
  const int64_t s = a.slots[i], before = i > 0 ? a.slots[i - 1] : -1;
  constexpr int kScan = static_cast<int>(kScanTokens) / kQThreads;
  int64_t all[kScan];
#pragma unroll
  for (int u = 0; u < kScan; ++u) {
    const int j = u * kQThreads + threadIdx.x;
    all[u] = j < a.n ? a.slots[j] : -1;
  }
  if (s < 0) return;  // padding row
  if (s >= a.num_slots) {
    if (threadIdx.x == 0 && blockIdx.y == 0) set_err(a.err, IR_DEVERR_SLOT);
    return;
  }
  const int64_t blk = static_cast<uint32_t>(s) / a.bs, lo = blk * a.bs;
  const int64_t near = before - lo;
  if (near >= 0 && near < a.bs) return;  // its neighbour or an earlier token owns the block
  for (int r = threadIdx.x; r < a.bs; r += kQThreads) src[r] = -1;
  __syncthreads();
  bool earlier = false;
#pragma unroll
  for (int u = 0; u < kScan; ++u) {
    const int j = u * kQThreads + threadIdx.x;
    const int64_t off = all[u] - lo;
    if (off < 0 || off >= a.bs) continue;
    earlier = earlier || j < i;
    atomicMax(&src[off], j);
  }
  if (__syncthreads_or(earlier)) return;
  const int task = blockIdx.y * kQWarps + (threadIdx.x >> 5);
  if (task < 2 * a.Hkv)
    quantise_task<T, C, VEC>(a, blk, [&](int r) { return src[r]; }, task / a.Hkv,
                             task % a.Hkv);
}

// Larger calls: the tokens' runs (neighbours in one block) are linked per
// block first. head[blk] is the block's last linked run + 1 (0: none), next[i]
// the run before it, owners[] the first linked run of every block, in the
// order they were found; count[0] is their number, count[1] that of the other
// runs (mostly 0: every block's rows are one run, and no list is read).
struct Q8Links {
  int* count;
  int* head;
  int* next;
  int* owners;
};

// (a kernel rather than a memset, so that the three grids can overlap their
// starts: 32768 rows 29.2 us from 29.9)
__global__ void fill_kernel(int* p, int n, int value) {
  let_next_grid_start();
  wait_prior_grid();
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x)
    p[i] = value;
}

__global__ void __launch_bounds__(kQThreads)
    link_runs_kernel(const int64_t* slots, int64_t n, int64_t num_slots, int bs, const Q8Links l,
                     int32_t* err) {
  __shared__ int found[kQWarps], base;
  let_next_grid_start();
  wait_prior_grid();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kQThreads + threadIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t s = i < n ? slots[i] : -1;
  const int64_t p = i > 0 && i < n ? slots[i - 1] : -1;
  bool owner = false;
  if (s >= num_slots) {
    set_err(err, IR_DEVERR_SLOT);
  } else if (s >= 0) {
    const int64_t blk = static_cast<uint32_t>(s) / bs;
    const int64_t off = p - blk * bs;
    if (off < 0 || off >= bs) {  // the first of its run
      const int prev = atomicExch(&l.head[blk], static_cast<int>(i) + 1);
      l.next[i] = prev;
      owner = prev == 0;
      if (!owner) atomicAdd(l.count + 1, 1);
    }
  }
  // one addition to the common count per CTA
  const unsigned m = __ballot_sync(kAll, owner);
  if (lane == 0) found[warp] = __popc(m);
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kQWarps; ++w) {
    before += w < warp ? found[w] : 0;
    all += found[w];
  }
  if (threadIdx.x == 0 && all > 0) base = atomicAdd(l.count, all);
  __syncthreads();
  if (owner) l.owners[base + before + __popc(m & ((1u << lane) - 1u))] = static_cast<int>(i);
}

// Calls f(in, offset, token) for the rows of the run that starts at `first`,
// then of the block's other runs, by one warp.
template <typename F>
__device__ __forceinline__ void walk_runs(const Q8WriteArgs& a, const Q8Links& l, int64_t blk,
                                          bool others, int first, F f) {
  const int lane = threadIdx.x & 31;
  const int64_t lo = blk * a.bs;
  for (int run = others ? l.head[blk] : first + 1; run != 0;) {
    const int64_t start = run - 1;
    run = others ? l.next[start] : 0;
    for (int64_t j = start + lane;; j += 32) {
      const int64_t off = j < a.n ? a.slots[j] - lo : -1;
      const bool in = off >= 0 && off < a.bs;
      // a run ends at its first token of another block
      const unsigned m = __ballot_sync(kAll, in);
      const int len = m == kAll ? 32 : __ffs(~m) - 1;
      f(lane < len, static_cast<int>(off), static_cast<int>(j));
      if (len < 32) break;
    }
  }
}

// Blocks of up to 32 rows: every warp takes a task of its own, lane r holding
// the token of row r.
template <typename T, typename C, bool VEC>
__global__ void __launch_bounds__(kQThreads, sizeof(T) == 2 ? 3 : 2)
    write_runs_kernel(const Q8WriteArgs a, const Q8Links l) {
  __shared__ int rows[kQWarps][32];
  wait_prior_grid();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // this warp's task of every `step`-th block
  const int tasks = 2 * a.Hkv, warps = gridDim.x * kQWarps;
  const int w = blockIdx.x * kQWarps + warp;
  const int step = warps / tasks, task = w % tasks;
  const int tside = task / a.Hkv, thead = task - tside * a.Hkv;
  const int count = w / tasks < step ? l.count[0] : 0;
  const bool others = l.count[1] != 0;
  int o = w / tasks;
  // the next block's first token and slots arrive during the current task
  int first = o < count ? l.owners[o] : 0;
  int next = step < count - o ? l.owners[o + step] : 0;
  auto slots_from = [&](int f) { return f + lane < a.n ? a.slots[f + lane] : -1; };
  int64_t mine = slots_from(first);
  for (; o < count; o += step) {
    const int64_t coming = slots_from(next);
    const int after = 2 * step < count - o ? l.owners[o + 2 * step] : 0;
    const uint32_t s0 = static_cast<uint32_t>(__shfl_sync(kAll, mine, 0));
    const int64_t blk = s0 / a.bs;
    const int64_t off = mine - blk * a.bs;
    // the run: up to its first token of another block
    const unsigned in = __ballot_sync(kAll, off >= 0 && off < a.bs);
    const int len = in == kAll ? 32 : __ffs(~in) - 1;
    const int off0 = __shfl_sync(kAll, static_cast<int>(off), 0);
    int row;  // token of row `lane`, or -1
    if (!others && len < 32 && __all_sync(kAll, lane >= len || off == off0 + lane)) {
      // rows in order
      row = lane >= off0 && lane < off0 + len ? first + lane - off0 : -1;
    } else {
      rows[warp][lane] = -1;
      __syncwarp();
      walk_runs(a, l, blk, others, first, [&](bool hit, int r, int j) {
        if (hit) atomicMax(&rows[warp][r], j);
      });
      __syncwarp();
      row = rows[warp][lane];
      __syncwarp();
    }
    quantise_task<T, C, VEC>(a, blk, [&](int r) { return __shfl_sync(kAll, row, r); }, tside,
                             thead);
    first = next;
    next = after;
    mine = coming;
  }
}

// A task with a value that is not finite, kept out of the common path's
// registers (row: token of block row `lane`).
template <typename T, typename C>
__device__ __noinline__ void quantise_apart(const Q8WriteArgs& a, int64_t blk, int row, int side,
                                            int h) {
  quantise_task<T, C, true>(a, blk, [&](int r) { return __shfl_sync(kAll, row, r & 31); }, side,
                            h);
}

// The same for 16-bit rows where a task's rows are at most one load of the
// warp (bs * D <= 2048): the rows of the next task are copied to shared memory
// while the current one is computed, so that a warp's reads never pause; every
// lane copies and reads its own pieces. Two CTAs fill an SM's registers (32768
// rows of 4 heads of 128, bf16, the three grids together: 24.4 us = 4.1 TB/s, against 29.2
// with the rows in registers).
template <typename T, typename C>
__global__ void __launch_bounds__(kQThreads, 2) write_stream_kernel(const Q8WriteArgs a,
                                                                    const Q8Links l) {
  __shared__ int rows[kQWarps][32];
  extern __shared__ __align__(16) uint4 stage[];  // [warp][2][kPass][32]
  wait_prior_grid();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tasks = 2 * a.Hkv, warps = gridDim.x * kQWarps;
  const int w = blockIdx.x * kQWarps + warp;
  const int step = warps / tasks, task = w % tasks;
  const int side = task / a.Hkv, h = task - side * a.Hkv;
  int o = w / tasks;
  const int count = o < step ? l.count[0] : 0;
  const bool others = l.count[1] != 0;
  if (o >= count) return;
  const int sh = a.D == 128 ? 4 : 3;  // log2 of the lanes per row
  const int rp = 32 >> sh;
  const int sub = lane >> sh, col = (lane & ((1 << sh) - 1)) * 8;
  const T* in = reinterpret_cast<const T*>(a.src[side]) + h * a.D + col;
  const int row_bytes = a.Hkv * a.D;
  uint4* mine = stage + warp * (2 * kPass * 32) + lane;

  struct Task {
    int64_t blk;
    int row;        // token of row `lane`, or -1
    float before;   // the scale
    uint32_t have;
  };
  auto slots_from = [&](int f) { return f + lane < a.n ? a.slots[f + lane] : -1; };
  // resolves a task and starts its copies into buffer `buf`
  auto start = [&](int first, int64_t slot, int buf) {
    Task t;
    t.blk = static_cast<uint32_t>(__shfl_sync(kAll, slot, 0)) / a.bs;
    t.before = a.scale[side][t.blk * a.Hkv + h];
    const int64_t off = slot - t.blk * a.bs;
    const unsigned inside = __ballot_sync(kAll, off >= 0 && off < a.bs);
    const int len = inside == kAll ? 32 : __ffs(~inside) - 1;
    const int off0 = __shfl_sync(kAll, static_cast<int>(off), 0);
    if (!others && len < 32 && __all_sync(kAll, lane >= len || off == off0 + lane)) {
      t.row = lane >= off0 && lane < off0 + len ? first + lane - off0 : -1;  // rows in order
    } else {
      rows[warp][lane] = -1;
      __syncwarp();
      walk_runs(a, l, t.blk, others, first, [&](bool hit, int r, int j) {
        if (hit) atomicMax(&rows[warp][r], j);
      });
      __syncwarp();
      t.row = rows[warp][lane];
      __syncwarp();
    }
    const int some = __reduce_max_sync(kAll, t.row);
    t.have = 0;
#pragma unroll
    for (int u = 0; u < kPass; ++u) {
      const int r = u * rp + sub;
      int tok = __shfl_sync(kAll, t.row, r & 31);
      if (r < a.bs && tok >= 0)
        t.have |= 1u << u;
      else
        tok = some;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                       smem_u32(mine + (buf * kPass + u) * 32)),
                   "l"(in + static_cast<int64_t>(tok) * a.stride[side])
                   : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    return t;
  };

  int first = l.owners[o];
  int next = step < count - o ? l.owners[o + step] : 0;
  Task cur = start(first, slots_from(first), 0);
  int64_t slot = slots_from(next);
  for (int buf = 0;; buf ^= 1) {
    const bool more = step < count - o;
    Task coming;
    if (more) {
      coming = start(next, slot, buf ^ 1);
      next = 2 * step < count - o ? l.owners[o + 2 * step] : 0;
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    // (read twice, for the maximum and for the codes, not held in between)
    uint32_t m = 0;
#pragma unroll
    for (int u = 0; u < kPass; ++u) m = Eight<T>{mine[(buf * kPass + u) * 32]}.top(m);
    if (more) slot = slots_from(next);
    auto src = [&](int r) { return __shfl_sync(kAll, cur.row, r & 31); };
    const float amax = Eight<T>::magnitude(m);
    if (__any_sync(kAll, !finite(amax))) {
      quantise_apart<T, C>(a, cur.blk, cur.row, side, h);
    } else {
      const float top = __uint_as_float(__reduce_max_sync(kAll, __float_as_uint(amax)));
      const bool begun = src(0) >= 0;
      const float now = settle_scale<C>(top, false, begun, cur.before,
                                        a.scale[side] + cur.blk * a.Hkv + h);
      uint8_t* dst = a.pool[side] + cur.blk * a.bs * row_bytes + (h * a.D + col);
      const float inv = pow2_reciprocal(now);
      if (!begun && now != cur.before && now == now)
        rescale_rest<C>(a, src, dst, row_bytes, rp, sub, cur.before, now);
      uint8_t* to = dst + sub * row_bytes;
#pragma unroll 4
      for (int u = 0; u < kPass; ++u) {
        float v[8];
        Eight<T>{mine[(buf * kPass + u) * 32]}.values(v);
        if (inv != 0.f) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] *= inv;
        } else {  // a scale that is no power of two
          for (int i = 0; i < 8; ++i) v[i] = __fdiv_rn(v[i], now);
        }
        const uint2 c = encode8<C>(v);
        if ((cur.have >> u) & 1u) *reinterpret_cast<uint2*>(to + u * rp * row_bytes) = c;
      }
    }
    if (!more) return;
    cur = coming;
    o += step;
  }
}

// Larger blocks: a CTA per block, its rows' tokens in shared memory.
template <typename T, typename C, bool VEC>
__global__ void __launch_bounds__(kQThreads) write_blocks_kernel(const Q8WriteArgs a,
                                                                 const Q8Links l) {
  extern __shared__ int src[];
  wait_prior_grid();
  const int count = l.count[0];
  const bool others = l.count[1] != 0;
  const int warp = threadIdx.x >> 5;
  for (int o = blockIdx.x; o < count; o += gridDim.x) {
    const int first = l.owners[o];
    const int64_t blk = static_cast<uint32_t>(a.slots[first]) / a.bs;
    for (int r = threadIdx.x; r < a.bs; r += kQThreads) src[r] = -1;
    __syncthreads();
    if (warp == 0)
      walk_runs(a, l, blk, others, first, [&](bool in, int off, int j) {
        if (in) atomicMax(&src[off], j);
      });
    __syncthreads();
    for (int task = warp; task < 2 * a.Hkv; task += kQWarps)
      quantise_task<T, C, VEC>(a, blk, [&](int r) { return src[r]; }, task / a.Hkv,
                               task % a.Hkv);
    __syncthreads();
  }
}

// code * s beyond T's range saturates; a NaN code and a scale that is not finite
// keep their value.
template <typename T>
__device__ __forceinline__ float saturate(float x, float s) {
  constexpr float kTop = std::is_same<T, __half>::value ? 65504.f
                         : sizeof(T) == 2               ? 0x1.fep127f
                                                        : 0x1.fffffep127f;
  // (min and max would turn NaN into a number, the comparison keeps it)
  return fabsf(x) > kTop && finite(s) ? copysignf(kTop, x) : x;
}

// Whether any of four e4m3 codes is NaN (0x7f or 0xff).
__device__ __forceinline__ bool has_nan(uint32_t w) {
  // 0x7f + 1 carries into a byte's top bit, and nothing below it does
  return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0u;
}

// 8 codes to 8 values of T, likewise (out 16-byte aligned).
template <typename T, typename C>
__device__ __forceinline__ void store8(T* out, uint2 codes, float s) {
  const float4 f = decode4<C>(codes.x), g = decode4<C>(codes.y);
  const float v[8] = {saturate<T>(f.x * s, s), saturate<T>(f.y * s, s),
                      saturate<T>(f.z * s, s), saturate<T>(f.w * s, s),
                      saturate<T>(g.x * s, s), saturate<T>(g.y * s, s),
                      saturate<T>(g.z * s, s), saturate<T>(g.w * s, s)};
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(out)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(out)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(out) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]),
                                                pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  }
}

// 16 codes to 16 values of T, multiplied by the scale in fp32 and rounded once.
template <typename T, typename C>
__device__ __forceinline__ void store16(T* out, uint4 codes, float s, int vec) {
  constexpr float kLargest = std::is_same<C, int8_t>::value ? 127.f : 448.f;
  constexpr float kTop = std::is_same<T, __half>::value ? 65504.f : 3.38e38f;
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
  float v[16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 f = decode4<C>(w[i]);
    v[4 * i] = f.x * s, v[4 * i + 1] = f.y * s, v[4 * i + 2] = f.z * s, v[4 * i + 3] = f.w * s;
  }
  if (fabsf(s) > kTop / kLargest) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = saturate<T>(v[i], s);
  }
  if (!vec) {
#pragma unroll
    for (int i = 0; i < 16; ++i) out[i] = DT<T>::from_f(v[i]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<float4*>(out)[i] =
          make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      reinterpret_cast<uint4*>(out)[i] =
          make_uint4(pack2<T>(v[8 * i], v[8 * i + 1]), pack2<T>(v[8 * i + 2], v[8 * i + 3]),
                     pack2<T>(v[8 * i + 4], v[8 * i + 5]), pack2<T>(v[8 * i + 6], v[8 * i + 7]));
  }
}

// Threads that cover a row of this many pieces: as many rows side
// by side as a CTA holds, or the whole CTA in turns.
inline int piece_threads(int pieces) { return pieces >= 256 ? 256 : 256 / pieces * pieces; }

// Rows by slot; a thread reads the same piece of kRows rows at once (with more
// CTAs in flight one does best: both sides of 32768 rows of 4 heads of 128 to
// bf16, 101 MB, 23.7 us = 4.3 TB/s; 2 and 4 rows 24.2 and 25.5). Bound by the
// chain slot, then scale and codes, of one load a thread (HBM 14 % busy, the
// written rows stay in L2).
constexpr int kRows = 1;
template <typename T, typename C>
__global__ void __launch_bounds__(256)
    gather_q8_kernel(T* out, const uint8_t* pool, const float* scale, const int64_t* slots, int n,
                     int Hkv, int D, int bs, int shift, int64_t num_slots, int vec, int32_t* err) {
  wait_prior_grid();
  const int pieces = Hkv * D / 16;
  const int tpr = pieces < 256 ? pieces : 256;
  const int side = blockDim.x / tpr;  // rows side by side
  const int c0 = threadIdx.x % tpr;
  const int row0 = blockIdx.x * side * kRows + threadIdx.x / tpr;
  int64_t s[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) s[u] = row0 + u * side < n ? slots[row0 + u * side] : 0;
#pragma unroll
  for (int u = 0; u < kRows; ++u)
    if (s[u] < 0 || s[u] >= num_slots) {
      s[u] = -1;
      if (c0 == 0) set_err(err, IR_DEVERR_SLOT);
    }
  for (int c = c0; c < pieces; c += tpr) {
    const int h = c * 16 / D;
    uint4 codes[kRows];
    float sc[kRows];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const uint32_t at = s[u] < 0 ? 0u : static_cast<uint32_t>(s[u]);
      const uint32_t blk = shift >= 0 ? at >> shift : at / bs;
      codes[u] = reinterpret_cast<const uint4*>(pool)[static_cast<uint64_t>(at) * pieces + c];
      sc[u] = scale[static_cast<uint64_t>(blk) * Hkv + h];
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      if (s[u] < 0) codes[u] = make_uint4(0u, 0u, 0u, 0u), sc[u] = 0.f;
      if (row0 + u * side < n)
        store16<T, C>(out + (static_cast<int64_t>(row0 + u * side) * pieces + c) * 16, codes[u],
                      sc[u], vec);
    }
  }
}

// Whether one of 8 values code * s is lost as a row of fp16: beyond its range
// (where it would saturate), or, with `fine`, below its normal range and not a
// multiple of its smallest value. NaN is not: it stays NaN.
template <typename C>
__device__ __forceinline__ bool lost_in_half(uint2 codes, float s, bool fine) {
  bool lost = false;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 f = decode4<C>(i == 0 ? codes.x : codes.y);
    const float v[4] = {f.x * s, f.y * s, f.z * s, f.w * s};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      lost = lost || fabsf(v[e]) > 65504.f ||
             (fine && fabsf(v[e]) < 1.f && __half2float(__float2half_rn(v[e])) != v[e]);
  }
  return lost && finite(s);
}

// The blocks of the sequences' histories as rows of T: with `table` null, each
// in its own place of a pool laid out as the codes are; else sequence by
// sequence (cap rows each), with the block table of that order. The tensor
// cores multiply the masked weights of a key tile too, and 0 * NaN is NaN: a V
// that is not finite would reach rows that do not attend it. So it becomes 0,
// and its head's K NaN instead: the score of a row that attends it is NaN, and
// a masked score is never used.
//
// fp16 has fewer exponents than code * scale (bf16 has as many as fp32). Of the
// values that it cannot hold, a small V is off by at most 2^-25, half of the
// output's own smallest step; but a K or V beyond 65504 would saturate, and the
// error of a small K is multiplied by q, whatever its size. exact_from (fp16
// only) receives each sequence's first position with such a value, and behind
// the S sequences the smallest of all: rows from there on are left to the fp32
// kernel, which reads the codes. Powers of two in [2^-15, 2^7] (e4m3; int8
// [2^-24, 2^9]) have none, so the codes are looked at only under other scales. (A
// scale that is no power of two rounds a value to half a unit of T, as writing it
// to a 16-bit pool would.)
template <typename T, typename C>
__global__ void __launch_bounds__(256)
    expand_blocks_kernel(T* kout, T* vout, const uint8_t* kp, const uint8_t* vp, const float* ks,
                         const float* vs, const int32_t* bt, int64_t bt_stride, const int32_t* ctx,
                         const int32_t* q_start, int short_rows, int max_blocks,
                         int64_t num_blocks, int Hkv, int D, int bs, int32_t* table, int64_t cap,
                         int table_block, int32_t* exact_from, int32_t* err) {
  constexpr bool kHalfRows = std::is_same<T, __half>::value;
  constexpr bool kInt = std::is_same<C, int8_t>::value;
  constexpr float kFinest = kInt ? 0x1p-24f : 0x1p-15f;
  constexpr float kWidest = 65504.f / (kInt ? 127.f : 448.f);
  int first = INT32_MAX;  // first position that fp16 rows cannot hold
  wait_prior_grid();
  const int sq = blockIdx.x;
  // (sequences of few rows are attended from the codes)
  const int64_t c0 = q_start[sq + 1] - q_start[sq] > short_rows ? ctx[sq] : 0;
  const int pieces = Hkv * D / 8;
  const int tpr = pieces < 256 ? pieces : 256;
  const int side = blockDim.x / tpr;
  if (threadIdx.x == 0 && blockIdx.y == 0 && c0 > static_cast<int64_t>(max_blocks) * bs)
    set_err(err, IR_DEVERR_CONTEXT_LEN);
  for (int j = blockIdx.y; j < max_blocks && static_cast<int64_t>(j) * bs < c0; j += gridDim.y) {
    int64_t id = bt[sq * bt_stride + j];
    bool ok = id >= 0 && id < num_blocks;
    if (!ok) {
      // in place the attention kernel reports it and reads zeros
      if (table == nullptr) continue;
      if (threadIdx.x == 0) set_err(err, IR_DEVERR_BLOCK_ID);
      id = 0;
    }
    const int64_t to = table ? sq * cap + static_cast<int64_t>(j) * bs : id * bs;
    for (int c = threadIdx.x % tpr; c < pieces; c += tpr) {
      const float k = ok ? ks[id * Hkv + c * 8 / D] : 0.f, v = ok ? vs[id * Hkv + c * 8 / D] : 0.f;
      const bool fine = fabsf(k) < kFinest;
      const bool look = kHalfRows && (fine || fabsf(k) > kWidest || fabsf(v) > kWidest);
#pragma unroll 4
      for (int r = threadIdx.x / tpr; r < bs; r += side) {
        const int64_t at = (id * bs + r) * pieces + c, dst = (to + r) * pieces + c;
        uint2 kc = reinterpret_cast<const uint2*>(kp)[at];
        uint2 vc = reinterpret_cast<const uint2*>(vp)[at];
        if (!ok) kc = vc = make_uint2(0u, 0u);
        if (kHalfRows && look && j * bs + r < c0 &&
            (lost_in_half<C>(kc, k, fine) || lost_in_half<C>(vc, v, false)))
          first = min(first, j * bs + r);
        float kr = k, vr = v;
        if (!finite(v) || (std::is_same<C, e4m3_t>::value && (has_nan(vc.x) || has_nan(vc.y)))) {
          kr = __uint_as_float(0x7fc00000u);
          vr = 0.f;
          vc = make_uint2(0u, 0u);
        }
        store8<T, C>(kout + dst * 8, kc, kr);
        store8<T, C>(vout + dst * 8, vc, vr);
      }
    }
  }
  if (table != nullptr && blockIdx.y == 0)
    for (int i = threadIdx.x; i < cap / table_block; i += blockDim.x)
      table[sq * (cap / table_block) + i] = static_cast<int32_t>(sq * (cap / table_block) + i);
  if (kHalfRows && first != INT32_MAX) {
    atomicMin(&exact_from[sq], first);
    atomicMin(&exact_from[gridDim.x], first);
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

}  // namespace

size_t cache_write_q8_workspace(int64_t n, int64_t num_blocks) {
  if (n <= kScanTokens) return 0;
  const int64_t owners = n < num_blocks ? n : num_blocks;
  return align256(static_cast<size_t>(num_blocks + 2) * 4) + align256(static_cast<size_t>(n) * 4) +
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
  a.stride[0] = static_cast<int>(k_stride);
  a.stride[1] = static_cast<int>(v_stride);
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
  const bool vec = (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0 &&
                   (k_stride * eb) % 16 == 0 && (v_stride * eb) % 16 == 0;
  a.err = err;
  const size_t smem = static_cast<size_t>(bs) * 4;
  if (n <= kScanTokens) {
    const dim3 grid(static_cast<unsigned>(n), (2 * Hkv + kQWarps - 1) / kQWarps);
    return by_type(dtype, [&](auto t) {
      return by_format(fmt, [&](auto c) {
        using T = decltype(t);
        using C = decltype(c);
        return launch_behind(vec ? write_scan_kernel<T, C, true> : write_scan_kernel<T, C, false>,
                             grid, kQThreads, smem, stream, a);
      });
    });
  }
  const int64_t num_blocks = num_slots / bs;
  uint8_t* w = static_cast<uint8_t*>(ws);
  const size_t heads = align256(static_cast<size_t>(num_blocks + 2) * 4);
  Q8Links l;
  l.count = reinterpret_cast<int*>(w);
  l.head = l.count + 2;
  l.next = reinterpret_cast<int*>(w + heads);
  l.owners = reinterpret_cast<int*>(w + heads + align256(static_cast<size_t>(n) * 4));
  const int words = static_cast<int>(num_blocks + 2);
  int rc = launch_behind(fill_kernel, dim3(words < 65536 ? (words + 255) / 256 : 256), 256, 0,
                         stream, l.count, words, 0);
  if (rc) return rc;
  rc = launch_behind(link_runs_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), 256, 0,
                         stream, slots, n, num_slots, bs, l, err);
  if (rc) return rc;
  const int64_t blocks = n < num_blocks ? n : num_blocks;
  const bool small = bs <= 32;
  // (at least one warp for every task of a block)
  const int64_t least = (2 * Hkv + kQWarps - 1) / kQWarps;
  int64_t grid = small ? (blocks * 2 * Hkv + kQWarps - 1) / kQWarps : blocks;
  // (as many CTAs as fit at once)
  const bool stream16 = dtype != IR_DTYPE_F32 && vec && small && bs * D <= 2048;
  const int64_t most = static_cast<int64_t>(sms) * (dtype == IR_DTYPE_F32 || stream16 ? 2 : 3);
  if (grid > most) grid = most;
  if (small && grid < least) grid = least;
  return by_type(dtype, [&](auto t) {
    return by_format(fmt, [&](auto c) {
      using T = decltype(t);
      using C = decltype(c);
      if constexpr (sizeof(T) == 2) {
        if (stream16) {
          auto stream_kern = write_stream_kernel<T, C>;
          constexpr int kStage = kQWarps * 2 * kPass * 32 * 16;  // 64 KB
          cudaError_t e = cudaFuncSetAttribute(
              stream_kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kStage);
          if (e != cudaSuccess) return static_cast<int>(e);
          return launch_behind(stream_kern, dim3(static_cast<unsigned>(grid)), kQThreads, kStage,
                               stream, a, l);
        }
      }
      auto kern = small ? (vec ? write_runs_kernel<T, C, true> : write_runs_kernel<T, C, false>)
                        : (vec ? write_blocks_kernel<T, C, true> : write_blocks_kernel<T, C, false>);
      return launch_behind(kern, dim3(static_cast<unsigned>(grid)), kQThreads, small ? 0 : smem,
                           stream, a, l);
    });
  });
}

int launch_cache_gather_q8(void* out, const void* pool, const float* scale, const int64_t* slots,
                           int64_t n, int Hkv, int D, int bs, int64_t num_slots, int dtype,
                           int fmt, int32_t* err, cudaStream_t stream) {
  const int pieces = Hkv * D / 16, threads = piece_threads(pieces);
  const int64_t rows = static_cast<int64_t>(pieces < 256 ? threads / pieces : 1) * kRows;
  const int64_t grid = (n + rows - 1) / rows;
  const int vec = reinterpret_cast<uintptr_t>(out) % 16 == 0;
  int shift = 0;  // log2(bs), or -1
  while ((1 << shift) < bs && shift < 30) ++shift;
  if ((1 << shift) != bs) shift = -1;
  return by_type(dtype, [&](auto t) {
    return by_format(fmt, [&](auto c) {
      using T = decltype(t);
      return launch_behind(gather_q8_kernel<T, decltype(c)>, dim3(static_cast<unsigned>(grid)),
                           threads, 0, stream,
                           static_cast<T*>(out), static_cast<const uint8_t*>(pool), scale, slots,
                           static_cast<int>(n), Hkv, D, bs, shift, num_slots, vec, err);
    });
  });
}

int launch_expand_blocks(void* k_out, void* v_out, const void* k_pool, const void* v_pool,
                         const float* k_scale, const float* v_scale, const int32_t* bt,
                         int64_t bt_stride, const int32_t* ctx, const int32_t* q_start,
                         int short_rows, int S, int max_blocks, int64_t num_blocks, int Hkv,
                         int D, int bs, int dtype, int fmt, int32_t* table, int64_t cap,
                         int table_block, int32_t* exact_from, int32_t* err,
                         cudaStream_t stream) {
  if (S == 0 || max_blocks == 0) return 0;
  if (exact_from) {
    const int rc = launch_behind(fill_kernel, dim3(S < 65536 ? S / 256 + 1 : 256), 256, 0, stream,
                                 exact_from, S + 1, INT32_MAX);
    if (rc) return rc;
  }
  const dim3 grid(static_cast<unsigned>(S),
                  static_cast<unsigned>(max_blocks < 4096 ? max_blocks : 4096));
  return by_type(dtype, [&](auto t) {
    return by_format(fmt, [&](auto c) {
      using T = decltype(t);
      return launch_behind(expand_blocks_kernel<T, decltype(c)>, grid,
                           piece_threads(Hkv * D / 8), 0, stream, static_cast<T*>(k_out),
                           static_cast<T*>(v_out), static_cast<const uint8_t*>(k_pool),
                           static_cast<const uint8_t*>(v_pool), k_scale, v_scale, bt, bt_stride,
                           ctx, q_start, short_rows, max_blocks, num_blocks, Hkv, D, bs, table,
                           cap, table_block, exact_from, err);
    });
  });
}

}  // namespace irb
