// Paged decode attention over 8-bit pools (e4m3 or int8 codes, one scale per
// block and kv head): TMA-fed, warp-specialised, half the bytes of the 16-bit
// kernel per token.
//
// Work partition, pieces and merge are the 16-bit kernel's (decode_common.cuh).
// A CTA owns HG kv heads and one share of the 16-token tiles. The producer
// warp resolves 32 tiles at a time and sends items of up to W = kConsumers / HG
// neighbouring tiles of one sequence through a ring of stages; its lanes issue
// the tiles' tensor copies (one box per block and side: [HG][rows][D] bytes)
// and copy the blocks' scales with 4-byte asynchronous copies that complete on
// the same barrier. Consumer warp (head, w) takes tile w of every item, so
// that kConsumers warps work whatever the head count; at the end of a segment
// the W warps of a head combine their states through shared memory.
//
// Mathematics of a tile (16 tokens, one kv head, up to 8 query heads per set):
//   S^T[16 x 8] = K[16 x D] . Q^T     (codes as fp16, q as fp16)
//   s = S * (k scale of the block) * (2^-e of the q row) * softmax scale
//   O^T[D x 8]  = O^T * alpha + (v scale of the block) * (V^T . P^T)
// A code is exact in fp16. q is multiplied by a power of two that puts its
// row's largest magnitude in [2^13, 2^14), so its 8 (bf16) or 11 (fp16) bits
// stay exact down to 2^-27 of that. P is fp16 with exponents shifted by 2^7:
// one rounding of 2^-12 per weight, small weights kept down to 2^-31 of the
// largest. Scales are applied in fp32 to the fp32 accumulators, so they may
// have any value; the products P.V of one tile start from zero to keep the
// blocks' scales apart, at the cost of an FMA in place of the multiply that
// rescales the accumulator anyway.
//
// The tensor-core instructions are the warp-level form, as in the 16-bit
// kernel: 7 query heads per K/V byte stay far below the ridge, and the codes
// pass through registers to become fp16 operands. Which tokens and columns a
// lane holds is free as long as both products agree, so fragments come from
// 16-byte shared-memory reads of whole code words, without ldmatrix:
//   token of fragment row g: t(2p) = p, t(2p + 1) = 4 + (p ^ 1)
//   K: lane (g, q) reads the 16-byte chunks q, q + 4 of row t(g)
//   V: lane (g, q) reads D / 8 bytes of rows t(2q), t(2q + 1) (+ 8), and byte
//      pairs of two rows become the token pairs of the A operand
// t() makes every 8- or 16-lane phase of these reads touch each bank once
// under the 128-byte (D = 128) and the 64-byte (D = 64) swizzle.
#include "decode_common.cuh"
#include "kernels.h"
#include "quant.cuh"

namespace irb {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kConsumers = 8;             // consumer warps
constexpr int kThreads = 32 * (kConsumers + 1);
constexpr float kPShift = 7.f;            // P is scaled by 2^7

struct __align__(16) ItemQ8 {
  int b;
  int unit;
  int ntok;   // valid tokens of the item (16 per tile but the last)
  int flags;  // bits 0-7: tiles whose copies were issued
};
constexpr int kSegStart = 1 << 8;  // first item of a segment
constexpr int kWhole = 1 << 9;     // the segment is the whole sequence
constexpr int kEnd = 1 << 10;      // end-of-stream marker
constexpr int kQBuf1 = 1 << 11;    // the segment's q rows are in buffer 1

template <int D, int HG, int R, int NS, int NQ>
struct LayoutQ8 {
  static constexpr int W = kConsumers / HG;       // tiles per item
  static constexpr int NB = kTile / R;            // blocks per tile
  static constexpr int kRegion = R * D;           // one head of one box
  static constexpr int kBox = HG * kRegion;       // one box
  static constexpr int kSide = NB * kBox;         // K (or V) of one tile
  static constexpr int kTileBytes = 2 * kSide;
  static constexpr int kStage = W * kTileBytes;
  static constexpr int kScales = W * NB * 2 * HG;  // floats per stage
  static constexpr int off_scale = NS * kStage;
  static constexpr int off_desc = off_scale + NS * kScales * 4;
  static constexpr int off_bar = off_desc + NS * 16;  // full[NS], empty[NS], qfree[2], head[HG]
  static constexpr int off_misc = (off_bar + (2 * NS + 2 + HG) * 8 + 15) / 16 * 16;
  // misc: RangeInfo (64 B) + block-scan scratch; then (m, l) of every warp
  static constexpr int off_ml = off_misc + 64 + (kConsumers + 1) * 8 + 8;
  static constexpr int kMl = kConsumers * NQ * 8 * 2;  // floats
  static constexpr int kFlushStride = D + 4;
  static constexpr int kFlushFloats = NQ * 8 * kFlushStride;  // per consumer warp
  static constexpr int off_flush = (off_ml + kMl * 4 + 15) / 16 * 16;
  static constexpr int kQBuf = HG * NQ * 8 * D * 2;
  static constexpr int off_q = (off_flush + kConsumers * kFlushFloats * 4 + 127) / 128 * 128;
  static constexpr int kBytes = off_q + 2 * kQBuf;
  static constexpr int kAlloc = kBytes + 1024;  // slack for 1 KB alignment
};

// Stages that fit in one CTA's shared memory beside the other buffers.
template <int D, int HG, int R, int NQ>
constexpr int stages_q8() {
  using L0 = LayoutQ8<D, HG, R, 0, NQ>;
  constexpr int per = L0::kStage + L0::kScales * 4 + 16 + 16;
  constexpr int n = (227 * 1024 - L0::kAlloc - 256) / per;
  return n < 2 ? 2 : (n > 12 ? 12 : n);
}

// Four-byte asynchronous copy global -> shared, and this thread's arrival on
// `bar` once its earlier copies have landed (counted in the barrier's own
// expected arrivals).
__device__ __forceinline__ void copy4_async(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void arrive_after_copies(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

// Byte offset of 16-byte chunk c of row r (0..7 within its box's 8-row groups)
// in a region of D-byte rows under the copy's swizzle.
template <int D>
__device__ __forceinline__ int chunk_off(int r, int c) {
  return D == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}

template <typename T, typename C, int D, int HG, int R, int NQ, int NS>
__global__ void __launch_bounds__(kThreads, 1)
    decode_q8_kernel(const __grid_constant__ CUtensorMap tmk,
                     const __grid_constant__ CUtensorMap tmv, const DecodeArgs a, int q_bulk) {
  using L = LayoutQ8<D, HG, R, NS, NQ>;
  constexpr int W = L::W, NB = L::NB;
  constexpr int KS = D / 16;  // k-steps of Q.K, m-tiles of P.V
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int hgrp = blockIdx.x, g = blockIdx.y;
  const int kv0 = hgrp * HG;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::off_bar);
  uint64_t* empty = full + NS;
  uint64_t* qfree = empty + NS;
  uint64_t* hbar = qfree + 2;  // the W warps of a head meet here at a segment's end
  RangeInfo* ri = reinterpret_cast<RangeInfo*>(smem + L::off_misc);
  static_assert(sizeof(RangeInfo) <= 64, "RangeInfo fits its shared-memory slot");
  int64_t* sm_scan = reinterpret_cast<int64_t*>(smem + L::off_misc + 64);
  ItemQ8* desc = reinterpret_cast<ItemQ8*>(smem + L::off_desc);
  float* scales = reinterpret_cast<float*>(smem + L::off_scale);

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 33);  // the copies' byte count, and every producer lane
      mbar_init(&empty[i], kConsumers);
    }
    mbar_init(&qfree[0], kConsumers);
    mbar_init(&qfree[1], kConsumers);
    for (int i = 0; i < HG; ++i) mbar_init(&hbar[i], W);
    fence_mbar_init();
  }
  if (threadIdx.x == 32) {
    prefetch_tensormap(&tmk);
    prefetch_tensormap(&tmv);
  }
  wait_prerequisites();
  find_share<kThreads, T>(a, g, kv0, HG, ri, sm_scan);  // includes __syncthreads
  launch_dependents();
  const int64_t start = ri->start, end = ri->end;
  if (start >= end) return;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    int b = ri->b_first;
    int64_t pb = ri->p_first;
    int nb = tiles_of(a, b);
    int seg_base = 0;  // segments started before this batch
    uint32_t item = 0;
    bool abort = false;
    for (int64_t t = start; t < end && !abort;) {
      const int64_t tt = t + lane;
      const bool active = tt < end;
      int lb = b, ln = nb;
      int64_t lp = pb;
      if (active) {
        while (tt >= lp + ln) {
          lp += ln;
          ++lb;
          ln = tiles_of(a, lb);
        }
      }
      const int j = static_cast<int>(tt - lp);
      const int tok0 = j * kTile;
      int nvalid = 0, id0 = 0, id1 = -1, row0 = 0;
      bool ok = false, seg_start = false, whole = false;
      if (active) {
        nvalid = min(kTile, clamp_ctx(a.context_lens[lb], a) - tok0);
        const int32_t* btr = a.block_tables + lb * a.bt_stride;
        const int blk = tok0 / a.bs;
        id0 = btr[blk];
        ok = id0 >= 0 && id0 < a.num_blocks;
        row0 = id0 * a.bs + (tok0 - blk * a.bs);
        if (R == 8 && nvalid > 8) {
          id1 = btr[blk + 1];
          ok = ok && id1 >= 0 && id1 < a.num_blocks;
        }
        if (!ok) set_err(a.err, IR_DEVERR_BLOCK_ID);
        seg_start = (tt == start) || (j == 0);
        whole = (lp >= start) && (lp + ln <= end);
      }
      const unsigned starts = __ballot_sync(kFull, active && seg_start);
      const unsigned oks = __ballot_sync(kFull, ok);
      const int nact = (end - t) < 32 ? static_cast<int>(end - t) : 32;
      int k = 0;
      while (k < nact) {
        // tiles k .. k + n - 1: neighbours of one segment
        const unsigned later = starts & ~((2u << k) - 1u);
        const int lim = (k < 31 && later) ? __ffs(later) - 1 : nact;
        const int n = min(W, lim - k);
        if (n < W && lim == nact && t + nact < end && k > 0) break;  // look further first
        const uint32_t slot = item % NS;
        const uint32_t par = ((item / NS) & 1u) ^ 1u;
        const bool first = (starts >> k) & 1u;
        const int seg = seg_base + __popc(starts & ((2u << k) - 1u)) - 1;
        const bool with_q = q_bulk && first;
        int good = 1;
        if (lane == 0) {
          good = mbar_wait_bounded(&empty[slot], par) ? 1 : 0;
          if (good && with_q && seg >= 2)
            good = mbar_wait_bounded(&qfree[seg & 1], ((seg >> 1) + 1) & 1) ? 1 : 0;
        }
        if (!__shfl_sync(kFull, good, 0)) {
          if (lane == 0) set_err(a.err, IR_DEVERR_TIMEOUT);
          abort = true;
          break;
        }
        const int kb = __shfl_sync(kFull, lb, k);
        const int last_valid = __shfl_sync(kFull, nvalid, k + n - 1);
        const int kwhole = __shfl_sync(kFull, whole ? 1 : 0, k);
        const unsigned issued = (oks >> k) & ((1u << n) - 1u);
        uint8_t* st = smem + slot * L::kStage;
        if (lane == 0) {
          desc[slot] = ItemQ8{kb, g, (n - 1) * kTile + last_valid,
                              static_cast<int>(issued) | (first ? kSegStart : 0) |
                                  (kwhole ? kWhole : 0) | ((seg & 1) ? kQBuf1 : 0)};
          uint32_t bytes = 0;
          for (int w = 0; w < n; ++w)
            if ((issued >> w) & 1u)
              bytes += (R == 8 && w == n - 1 && last_valid <= 8) ? 2u * L::kBox
                                                                  : static_cast<uint32_t>(
                                                                        L::kTileBytes);
          const uint32_t qrows = static_cast<uint32_t>(HG * a.n_rep * D * 2);
          mbar_arrive_expect_tx(&full[slot], bytes + (with_q ? qrows : 0u));
          if (with_q)
            bulk_load(smem + L::off_q + (seg & 1) * L::kQBuf,
                      reinterpret_cast<const T*>(a.q) + kb * a.q_stride +
                          static_cast<int64_t>(kv0 * a.n_rep) * D,
                      qrows, &full[slot]);
        }
        __syncwarp();
        if (lane >= k && lane < k + n && ok) {
          uint8_t* td = st + (lane - k) * L::kTileBytes;
          tma_load_3d(td, &tmk, &full[slot], 0, row0, kv0);
          tma_load_3d(td + L::kSide, &tmv, &full[slot], 0, row0, kv0);
          if (R == 8 && id1 >= 0) {
            tma_load_3d(td + L::kBox, &tmk, &full[slot], 0, id1 * a.bs, kv0);
            tma_load_3d(td + L::kSide + L::kBox, &tmv, &full[slot], 0, id1 * a.bs, kv0);
          }
        }
        // scales[tile][block][side][head]
        float* sc = scales + slot * L::kScales;
#pragma unroll
        for (int base = 0; base < L::kScales; base += 32) {
          const int i = base + lane;
          const int w = i / (NB * 2 * HG), rem = i % (NB * 2 * HG);
          const int blk = rem / (2 * HG), side = rem / HG % 2, h = rem % HG;
          const int src = (k + w) & 31;
          const int i0 = __shfl_sync(kFull, id0, src), i1 = __shfl_sync(kFull, id1, src);
          const int id = blk == 0 ? i0 : i1;
          if (i < L::kScales && w < n && ((issued >> w) & 1u) && id >= 0)
            copy4_async(sc + i, (side ? a.v_scale : a.k_scale) +
                                    static_cast<int64_t>(id) * a.Hkv + kv0 + h);
        }
        arrive_after_copies(&full[slot]);
        ++item;
        k += n;
      }
      if (abort) break;
      seg_base += __popc(starts & (k >= 32 ? kFull : ((1u << k) - 1u)));
      // the cursor at the last tile issued
      b = __shfl_sync(kFull, lb, k - 1);
      pb = __shfl_sync(kFull, lp, k - 1);
      nb = __shfl_sync(kFull, ln, k - 1);
      t += k;
    }
    if (!abort) {
      const uint32_t slot = item % NS;
      const uint32_t par = ((item / NS) & 1u) ^ 1u;
      int good = 1;
      if (lane == 0) good = mbar_wait_bounded(&empty[slot], par) ? 1 : 0;
      if (__shfl_sync(kFull, good, 0)) {
        if (lane == 0) {
          desc[slot] = ItemQ8{0, 0, 0, kEnd};
          mbar_arrive(&full[slot]);
        }
        __syncwarp();
        mbar_arrive(&full[slot]);
      } else if (lane == 0) {
        set_err(a.err, IR_DEVERR_TIMEOUT);
      }
    }
    return;
  }

  // -------------------------------------------------------------- consumers
  const int cw = warp - 1;
  const int head = cw / W, w = cw % W;
  const int kvh = kv0 + head;
  const int grp = lane >> 2, qq = lane & 3, qd = qq * 2;
  const int tg = (grp & 1) ? 4 + ((grp >> 1) ^ 1) : grp >> 1;  // token of fragment row grp
  // byte offsets of this lane's reads within one 8-row half of a region
  int koff[D / 64];
#pragma unroll
  for (int c = 0; c < D / 64; ++c) koff[c] = chunk_off<D>(tg, qq + 4 * c);
  const int ta = qq, tb = 4 + (qq ^ 1);  // tokens of fragment rows 2 qq, 2 qq + 1
  // V columns of this lane: D / 8 bytes, piece `pc` of the row
  const int pc = D == 128 ? ((grp & 1) << 2) | (grp >> 1)
                          : ((((grp >> 1) & 1) << 1 | (grp >> 2)) << 1) | (grp & 1);
  const int va = D == 128 ? chunk_off<D>(ta, pc) : chunk_off<D>(ta, pc >> 1) + (pc & 1) * 8;
  const int vb = D == 128 ? chunk_off<D>(tb, pc) : chunk_off<D>(tb, pc >> 1) + (pc & 1) * 8;
  // second half of a tile: 8 rows on in the same box, or the second box
  constexpr int kHalf = R == 8 ? L::kBox : 8 * D;

  float acc[NQ][KS][4];
  float m[NQ][2], l[NQ][2], qinv[NQ][2];
  uint32_t qf[NQ][KS][2];
  auto reset = [&]() {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int i = 0; i < KS; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }
  };
  reset();
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    qinv[n][0] = qinv[n][1] = 0.f;
#pragma unroll
    for (int i = 0; i < KS; ++i) qf[n][i][0] = qf[n][i][1] = 0u;
  }
  int seg_b = -1, seg_unit = 0;
  bool seg_whole = false, have_seg = false;
  uint32_t meets = 0;  // phases of hbar passed
  float* ml = reinterpret_cast<float*>(smem + L::off_ml);
  float* fl = reinterpret_cast<float*>(smem + L::off_flush) + cw * L::kFlushFloats;

  // The W warps of this head wait for one another (bounded).
  auto meet = [&]() {
    if (W == 1) {
      __syncwarp();
      return true;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&hbar[head]);
    const bool ok = mbar_wait_bounded(&hbar[head], meets & 1u);
    ++meets;
    return __all_sync(kFull, ok) != 0;
  };

  // Combine the W states of the finished segment and write its rows: the
  // output (whole sequences) or a normalised fp32 piece.
  auto flush = [&]() {
    const int nr = a.n_rep;
    const int64_t pslot = static_cast<int64_t>(kvh) * a.ws_slots + seg_unit + seg_b;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        float x = l[n][jj];
        x += __shfl_xor_sync(kFull, x, 4);
        x += __shfl_xor_sync(kFull, x, 8);
        x += __shfl_xor_sync(kFull, x, 16);
        l[n][jj] = x;
        if (grp == 0) {
          float* p = ml + ((cw * NQ + n) * 8 + qd + jj) * 2;
          p[0] = m[n][jj];
          p[1] = x;
        }
      }
    if (!meet()) return false;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        float M = -INFINITY;
#pragma unroll
        for (int i = 0; i < W; ++i)
          M = fmaxf(M, ml[(((head * W + i) * NQ + n) * 8 + qd + jj) * 2]);
        const float use = M == -INFINITY ? 0.f : M;
        float Ls = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float* p = ml + (((head * W + i) * NQ + n) * 8 + qd + jj) * 2;
          Ls += p[1] * ex2(p[0] - use);
        }
        // nothing attended: zero (a NaN sum is not nothing)
        const float f = Ls == 0.f ? 0.f : ex2(m[n][jj] - use) / Ls;
        float* row = fl + (n * 8 + qd + jj) * L::kFlushStride + pc * (D / 8);
#pragma unroll
        for (int i = 0; i < KS; i += 2)
          *reinterpret_cast<float4*>(row + 2 * i) =
              make_float4(acc[n][i][jj] * f, acc[n][i][jj + 2] * f, acc[n][i + 1][jj] * f,
                          acc[n][i + 1][jj + 2] * f);
      }
    if (!seg_whole && w == 0 && lane < nr) {
      // (read here: past the second meeting a faster warp may be at the next
      // segment's end)
      float M = -INFINITY;
#pragma unroll
      for (int i = 0; i < W; ++i)
        M = fmaxf(M, ml[(((head * W + i) * NQ) * 8 + lane) * 2]);
      const float use = M == -INFINITY ? 0.f : M;
      float Ls = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float* p = ml + (((head * W + i) * NQ) * 8 + lane) * 2;
        Ls += p[1] * ex2(p[0] - use);
      }
      a.ws_lse[pslot * nr + lane] = Ls == 0.f ? -INFINITY : use + log2f(Ls) - kPShift;
    }
    if (!meet()) return false;
    const float* f0 = reinterpret_cast<const float*>(smem + L::off_flush) +
                      head * W * L::kFlushFloats;
    constexpr int kPer = D / 8;
    for (int c = w * 32 + lane; c < nr * kPer; c += 32 * W) {
      const int n = c / kPer, d = (c % kPer) * 8;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float* p = f0 + i * L::kFlushFloats + n * L::kFlushStride + d;
        const float4 u = *reinterpret_cast<const float4*>(p);
        const float4 v = *reinterpret_cast<const float4*>(p + 4);
        x.x += u.x, x.y += u.y, x.z += u.z, x.w += u.w;
        y.x += v.x, y.y += v.y, y.z += v.z, y.w += v.w;
      }
      if (seg_whole) {
        T* dst = reinterpret_cast<T*>(a.out) + seg_b * a.out_stride +
                 static_cast<int64_t>(kvh * nr + n) * D + d;
        *reinterpret_cast<uint4*>(dst) = make_uint4(pack2<T>(x.x, x.y), pack2<T>(x.z, x.w),
                                                    pack2<T>(y.x, y.y), pack2<T>(y.z, y.w));
      } else {
        float* dst = a.ws_o + (pslot * nr + n) * D + d;
        *reinterpret_cast<float4*>(dst) = x;
        *reinterpret_cast<float4*>(dst + 4) = y;
      }
    }
    if (W == 1) __syncwarp();
    reset();
    return true;
  };

  for (uint32_t item = 0;; ++item) {
    const uint32_t slot = item % NS, par = (item / NS) & 1u;
    const bool okw = mbar_wait_bounded(&full[slot], par);
    if (__any_sync(kFull, !okw)) {
      if (lane == 0) set_err(a.err, IR_DEVERR_TIMEOUT);
      break;
    }
    const ItemQ8 it = desc[slot];
    if ((it.flags & (kSegStart | kEnd)) && have_seg) {
      if (!flush()) {
        if (lane == 0) set_err(a.err, IR_DEVERR_TIMEOUT);
        break;
      }
    }
    if (it.flags & kEnd) break;
    if (it.flags & kSegStart) {
      have_seg = true;
      seg_b = it.b;
      seg_unit = it.unit;
      seg_whole = (it.flags & kWhole) != 0;
      const int buf = (it.flags & kQBuf1) ? 1 : 0;
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int hr = n * 8 + grp;  // query head of the group
        float v[D / 4];
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
          for (int e = 0; e < 16; ++e) v[c * 16 + e] = 0.f;
        if (hr < a.n_rep) {
          if (q_bulk) {
            const uint4* src = reinterpret_cast<const uint4*>(
                smem + L::off_q + buf * L::kQBuf + (head * a.n_rep + hr) * D * 2);
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const uint4 x = src[(qq + 4 * c) * 2 + u];
                const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float2 f = unpack2<T>(xs[e]);
                  v[c * 16 + u * 8 + 2 * e] = f.x;
                  v[c * 16 + u * 8 + 2 * e + 1] = f.y;
                }
              }
          } else {
            const T* src = reinterpret_cast<const T*>(a.q) + it.b * a.q_stride +
                           static_cast<int64_t>(kvh * a.n_rep + hr) * D;
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
              for (int e = 0; e < 16; ++e) v[c * 16 + e] = DT<T>::to_f(src[(qq + 4 * c) * 16 + e]);
          }
        }
#pragma unroll
        for (int e = 0; e < D / 4; ++e) top = fmaxf(top, fabsf(v[e]));
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
        // 2^(13 - floor(log2 top)), exponents kept where both factors are normal
        int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;
        ex = ex < -100 ? -100 : (ex > 126 ? 126 : ex);
        const float up = __uint_as_float(static_cast<uint32_t>(13 - ex + 127) << 23);
        const float down = __uint_as_float(static_cast<uint32_t>(ex - 13 + 127) << 23);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          const int o = (i >> 2) * 16 + (i & 3) * 4;
          qf[n][i][0] = pack2<__half>(v[o] * up, v[o + 1] * up);
          qf[n][i][1] = pack2<__half>(v[o + 2] * up, v[o + 3] * up);
        }
        const float inv = down * a.scale_log2;
        qinv[n][0] = __shfl_sync(kFull, inv, qd * 4);
        qinv[n][1] = __shfl_sync(kFull, inv, (qd + 1) * 4);
      }
      if (q_bulk) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&qfree[buf]);
      }
    }
    const int nvalid = ((it.flags >> w) & 1) ? min(kTile, it.ntok - w * kTile) : 0;
    if (nvalid > 0) {
      const uint32_t kbase = smem_u32(smem + slot * L::kStage + w * L::kTileBytes) +
                             head * L::kRegion;
      const uint32_t vbase = kbase + L::kSide;
      const float* sc = scales + slot * L::kScales + w * (NB * 2 * HG) + head;
      // scales of the tile's first and second 8 tokens
      const float ks0 = sc[0], vs0 = sc[HG];
      const float ks1 = NB == 2 ? (nvalid > 8 ? sc[2 * HG] : 0.f) : ks0;
      const float vs1 = NB == 2 ? (nvalid > 8 ? sc[3 * HG] : 0.f) : vs0;

      // V codes early: their reads overlap the score product
      constexpr int VW = D / 32;  // words per lane and token
      uint32_t vw[4][VW];
      {
        const uint32_t at[4] = {vbase + va, vbase + vb, vbase + kHalf + va, vbase + kHalf + vb};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (D == 128) {
            const uint4 x = lds128(at[i]);
            vw[i][0] = x.x, vw[i][1] = x.y, vw[i][2] = x.z, vw[i][3] = x.w;
          } else {
            const uint2 x = lds64(at[i]);
            vw[i][0] = x.x, vw[i][1] = x.y;
          }
        }
        if (nvalid < kTile) {
          // rows past the context may hold NaN codes, and 0 * NaN is NaN
          const int tk[4] = {ta, tb, ta + 8, tb + 8};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (tk[i] >= nvalid) {
#pragma unroll
              for (int e = 0; e < VW; ++e) vw[i][e] = 0u;
            }
        }
      }

      float s[NQ][4];
#pragma unroll
      for (int n = 0; n < NQ; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const uint4 x = lds128(kbase + koff[c]), y = lds128(kbase + kHalf + koff[c]);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t a0, a1, a2, a3;
          decode4_h<C>(xs[e], a0, a2);
          decode4_h<C>(ys[e], a1, a3);
#pragma unroll
          for (int n = 0; n < NQ; ++n)
            mma_16816<__half>(s[n], a0, a1, a2, a3, qf[n][c * 4 + e][0], qf[n][c * 4 + e][1]);
        }
      }

      const bool v0 = tg < nvalid, v1 = tg + 8 < nvalid;
      uint32_t pb0[NQ], pb1[NQ];
      float alpha[NQ][2];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float p[4];
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
          const float s0 = v0 ? s[n][jj] * (qinv[n][jj] * ks0) : -INFINITY;
          const float s1 = v1 ? s[n][jj + 2] * (qinv[n][jj] * ks1) : -INFINITY;
          float mx = fmaxf(s0, s1);
          mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, 16));
          const float mnew = fmaxf(m[n][jj], mx);
          const float muse = (mnew == -INFINITY) ? 0.f : mnew;
          alpha[n][jj] = ex2(m[n][jj] - muse);
          p[jj] = ex2(s0 - muse + kPShift);
          p[jj + 2] = ex2(s1 - muse + kPShift);
          l[n][jj] = l[n][jj] * alpha[n][jj] + p[jj] + p[jj + 2];
          m[n][jj] = mnew;
        }
        pb0[n] = movmatrix_trans(pack2<__half>(p[0], p[1]));
        pb1[n] = movmatrix_trans(pack2<__half>(p[2], p[3]));
      }

      // O^T = O^T * alpha + vs * (V^T . P^T)
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        uint32_t a0[2], a1[2], a2[2], a3[2];
        decode4_h<C>(__byte_perm(vw[0][e], vw[1][e], 0x5140), a0[0], a1[0]);
        decode4_h<C>(__byte_perm(vw[0][e], vw[1][e], 0x7362), a0[1], a1[1]);
        decode4_h<C>(__byte_perm(vw[2][e], vw[3][e], 0x5140), a2[0], a3[0]);
        decode4_h<C>(__byte_perm(vw[2][e], vw[3][e], 0x7362), a2[1], a3[1]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            float* o = acc[n][2 * e + u];
            if (NB == 1) {
              float x[4] = {0.f, 0.f, 0.f, 0.f};
              mma_16816<__half>(x, a0[u], a1[u], a2[u], a3[u], pb0[n], pb1[n]);
#pragma unroll
              for (int i = 0; i < 4; ++i) o[i] = fmaf(vs0, x[i], o[i] * alpha[n][i & 1]);
            } else {
              // two blocks: their products apart
              float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
              mma_16816<__half>(x, a0[u], a1[u], a2[u], a3[u], pb0[n], 0u);
              mma_16816<__half>(y, a0[u], a1[u], a2[u], a3[u], 0u, pb1[n]);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                o[i] = fmaf(vs1, y[i], fmaf(vs0, x[i], o[i] * alpha[n][i & 1]));
            }
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[slot]);
  }
}

// ---------------------------------------------------------------- dispatch

struct CallQ8 {
  const CUtensorMap *tmk, *tmv;
  const DecodeArgs* a;
  int q_bulk;
  cudaStream_t s;
};

template <typename T, typename C, int D, int HG, int R, int NQ>
int run_q8(const CallQ8* call) {
  constexpr int NS = stages_q8<D, HG, R, NQ>();
  using L = LayoutQ8<D, HG, R, NS, NQ>;
  static_assert(L::kAlloc <= 227 * 1024, "shared memory budget");
  static_assert(NQ * 8 * 2 <= 32, "one lane per query head of a group");
  auto kern = decode_q8_kernel<T, C, D, HG, R, NQ, NS>;
  cudaError_t e =
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kAlloc);
  if (e != cudaSuccess) return static_cast<int>(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(call->a->Hkv / HG, call->a->G);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::kAlloc;
  cfg.stream = call->s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return static_cast<int>(
      cudaLaunchKernelEx(&cfg, kern, *call->tmk, *call->tmv, *call->a, call->q_bulk));
}

template <typename T, typename C, int D, int HG, int NQ>
int by_rows(const CallQ8* c) {
  return c->a->bs == 8 ? run_q8<T, C, D, HG, 8, NQ>(c) : run_q8<T, C, D, HG, 16, NQ>(c);
}
template <typename T, typename C, int D>
int by_heads(const CallQ8* c) {
  const int hg = q8_head_group(c->a->Hkv, c->a->n_rep);
  if (c->a->n_rep <= 8) {
    switch (hg) {
      case 1: return by_rows<T, C, D, 1, 1>(c);
      case 2: return by_rows<T, C, D, 2, 1>(c);
      case 4: return by_rows<T, C, D, 4, 1>(c);
      default: return by_rows<T, C, D, 8, 1>(c);
    }
  }
  switch (hg) {
    case 1: return by_rows<T, C, D, 1, 2>(c);
    case 2: return by_rows<T, C, D, 2, 2>(c);
    default: return by_rows<T, C, D, 4, 2>(c);
  }
}
template <typename T, typename C>
int by_dim(const CallQ8* c) {
  return c->a->D == 128 ? by_heads<T, C, 128>(c) : by_heads<T, C, 64>(c);
}
template <typename T>
int by_code(int fmt, const CallQ8* c) {
  return fmt == IR_KV_INT8 ? by_dim<T, int8_t>(c) : by_dim<T, e4m3_t>(c);
}

}  // namespace

int q8_head_group(int num_kv_heads, int n_rep) {
  for (int hg : {8, 4, 2})
    if (num_kv_heads % hg == 0 && (hg < 8 || n_rep <= 8)) return hg;
  return 1;
}

int launch_decode_q8(const CUtensorMap& tmk, const CUtensorMap& tmv, const DecodeArgs& a,
                     int dtype, int fmt, cudaStream_t stream) {
  // q rows of a head group move as one bulk copy when 16-byte aligned
  const int q_bulk = reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && (a.q_stride * 2) % 16 == 0;
  const CallQ8 call{&tmk, &tmv, &a, q_bulk, stream};
  return dtype == IR_DTYPE_BF16 ? by_code<__nv_bfloat16>(fmt, &call)
                                : by_code<__half>(fmt, &call);
}

}  // namespace irb
