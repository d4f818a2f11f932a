// Paged decode attention over 8-bit pools (e4m3 or int8 codes, one scale per
// block and kv head): TMA-fed, warp-specialised, half the bytes of the 16-bit
// kernel per token.
//
// Work partition and pieces are the 16-bit kernel's (decode_common.cuh). A CTA
// owns HG kv heads and one share of the 16-token tiles. The producer warp
// resolves 32 tiles at a time, a lane each: sequence, block and scales. Items
// are up to W neighbouring tiles of one sequence and travel through a ring of
// stages; a tile's lane issues its tensor copies (one box per block and side:
// [HG][rows][D] bytes) and stores its scales beside them. 8 consumer warps share
// an item: WT = 8 / HG of them hold a state of each head (8 / (2 HG) for groups
// of 9-16 query heads, which make two sets of 8 with states of their own), and a
// warp takes tiles w and w + WT of the W = 2 WT together, since the work on a
// tile is a chain of dependent steps (blocks of 8 rows: one, a second set of
// scales takes the registers). 16 warps of half the registers spilled and were
// slower. At the end of a segment the warps of a state are combined through
// shared memory, in halves.
//
// Bound by HBM and by fixed costs: 64 sequences of 512-4096 tokens, 28 / 4 heads
// of 128, e4m3 (163 MB): 38.1 us = 4.3 TB/s; 4 of 32768, int8 (134 MB): 31.3 us.
// Without the arithmetic the same copies take 35.1; at the copy rate the bytes
// alone would take 25.5 and 20.8. Around the stream stand finding the share (1.3),
// the first tiles' tables (2.4), the first bytes (4.8), the CTAs' different ends
// (half of them have ended at 28, the last at 34), the last flush (1.4) and the
// merge (2.5).
// Short contexts (q8_seq_heads) have a CTA per sequence instead, without the
// first and the last of these: one of 201 tokens, int8, 2 heads of 64, 5.5 us.
//
// Mathematics of a tile (16 tokens, one kv head, 8 query heads):
//   S^T[16 x 8] = K[16 x D] . Q^T     (codes as fp16, q as fp16)
//   s = S * (k scale of the block) * (2^-e of the q row) * softmax scale
//   O^T[D x 8] += (v scale of the block) * (V^T . P^T),  P = 2^(s - m + 7)
// A code is exact in fp16. q is multiplied by a power of two that puts its
// row's largest magnitude in [2^13, 2^14), so its 8 (bf16) or 11 (fp16) bits
// stay exact down to 2^-27 of that. The reference m of a row is raised, and O
// rescaled, only when a score exceeds it by more than 8: P stays below 2^15,
// in fp16 with one rounding of 2^-11 per weight, and weights down to 2^-29 of
// the largest keep a nonzero value. Scales are applied in fp32 to the fp32
// accumulators, so they may have any value; the products P.V of one tile
// start from zero to keep the blocks' scales apart.
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
#include <atomic>

#include "decode_common.cuh"
#include "kernels.h"
#include "quant.cuh"

namespace irb {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kConsumers = 8;      // consumer warps
constexpr int kThreads = 32 * (kConsumers + 1);
constexpr float kPShift = 7.f;     // P is scaled by 2^7
constexpr float kSlack = 8.f;      // scores may exceed their row's reference by this

struct __align__(16) ItemQ8 {
  int b;
  int unit;
  int ntok;   // valid tokens of the item (16 per tile but the last)
  int flags;  // bits 0-15: tiles whose copies were issued
};
constexpr int kSegStart = 1 << 16;  // first item of a segment
constexpr int kWhole = 1 << 17;     // the segment is the whole sequence
constexpr int kEnd = 1 << 18;       // end-of-stream marker
constexpr int kQBuf1 = 1 << 19;     // the segment's q rows are in buffer 1

// SETS: a group of 9-16 query heads, as two sets of 8 with a state each.
template <int D, int HG, int R, int NS, bool SETS>
struct LayoutQ8 {
  static constexpr int kRows = SETS ? 2 * HG : HG;   // (head, query set) pairs
  static constexpr int WT = kConsumers / kRows;      // warps that share a pair's state
  // tiles a warp takes of an item at once (of 8-row blocks one: their second
  // set of scales and products takes the place)
  static constexpr int kPair = R == 8 ? 1 : 2;
  static constexpr int W = WT * kPair;               // tiles per item
  static constexpr int NB = kTile / R;            // blocks per tile
  static constexpr int kRegion = R * D;           // one head of one box
  static constexpr int kBox = HG * kRegion;       // one box
  static constexpr int kSide = NB * kBox;         // K (or V) of one tile
  static constexpr int kTileBytes = 2 * kSide;
  static constexpr int kStage = W * kTileBytes;
  static constexpr int kScales = W * NB * 2 * HG;  // floats per stage
  static constexpr int off_scale = NS * kStage;
  static constexpr int off_desc = off_scale + NS * kScales * 4;
  // full[NS], empty[NS], qfree[2], then one per consumer warp (see the flush)
  static constexpr int off_bar = off_desc + NS * 16;
  static constexpr int off_misc = (off_bar + (2 * NS + 2 + kConsumers) * 8 + 15) / 16 * 16;
  // misc: RangeInfo (64 B) + block-scan scratch; then (m, l) of every warp
  static constexpr int off_ml = off_misc + 64 + (kConsumers + 1) * 8 + 8;
  static constexpr int kMl = kConsumers * 8 * 2;
  static constexpr int kPart = 8 * D;             // floats of one warp's O
  static constexpr int off_part = (off_ml + kMl * 4 + 15) / 16 * 16;
  static constexpr int kParts = kRows * (WT / 2);
  static constexpr int off_q = (off_part + kParts * kPart * 4 + 127) / 128 * 128;
  // q rows of the current and the next segment: the group's own size, so that
  // the merge kernel's CTAs mostly find room beside this kernel's
  static constexpr int kAlloc = off_q + 2 * HG * (SETS ? 16 : 8) * D * 2;  // at most
  static int bytes(int n_rep) { return off_q + 2 * HG * n_rep * D * 2; }
};

// Stages that fit in one CTA's shared memory beside the other buffers.
template <int D, int HG, int R, bool SETS, int NS = 12>
constexpr int stages_q8() {
  if constexpr (NS == 2 || LayoutQ8<D, HG, R, NS, SETS>::kAlloc <= 227 * 1024)
    return NS;
  else
    return stages_q8<D, HG, R, SETS, NS - 1>();
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

template <typename T, typename C, int D, int HG, int R, bool SETS, int NS>
__global__ void __launch_bounds__(kThreads, 1)
    decode_q8_kernel(const __grid_constant__ CUtensorMap tmk,
                     const __grid_constant__ CUtensorMap tmv, const DecodeArgs a, int q_bulk) {
  using L = LayoutQ8<D, HG, R, NS, SETS>;
  constexpr int W = L::W, NB = L::NB, WT = L::WT, kPair = L::kPair;
  constexpr int KS = D / 16;  // k-steps of Q.K, m-tiles of P.V
  extern __shared__ __align__(1024) uint8_t smem[];  // (the swizzles count from here)
  const int hgrp = blockIdx.x, g = blockIdx.y;
  const int kv0 = hgrp * HG;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::off_bar);
  uint64_t* empty = full + NS;
  uint64_t* qfree = empty + NS;
  uint64_t* hbar = qfree + 2;  // one per consumer warp
  RangeInfo* ri = reinterpret_cast<RangeInfo*>(smem + L::off_misc);
  static_assert(sizeof(RangeInfo) <= 64, "RangeInfo fits its shared-memory slot");
  int64_t* sm_scan = reinterpret_cast<int64_t*>(smem + L::off_misc + 64);
  ItemQ8* desc = reinterpret_cast<ItemQ8*>(smem + L::off_desc);
  float* scales = reinterpret_cast<float*>(smem + L::off_scale);

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kConsumers);
    }
    mbar_init(&qfree[0], kConsumers);
    mbar_init(&qfree[1], kConsumers);
    // a state's first warp: its buffers are free; the others: its O is written
    for (int i = 0; i < kConsumers; ++i) mbar_init(&hbar[i], i % WT == 0 && WT > 1 ? WT / 2 : 1);
    fence_mbar_init();
  }
  if (threadIdx.x == 32) {
    prefetch_tensormap(&tmk);
    prefetch_tensormap(&tmv);
  }
  __syncthreads();  // the barriers are set up
  const int q_buf = HG * a.n_rep * D * 2;  // bytes of one q buffer
  wait_prerequisites();
  launch_dependents();
  // The share of this CTA. Batches of up to 256 sequences: by the producer
  // alone, 8 sequences a lane, without a block-wide scan (the merge kernel sums
  // the tile prefix itself then); the rows of empty sequences by the others.
  constexpr int kEach = 8;
  if (a.per_seq) {
    if (warp == 0) {
      const int c = a.context_lens[g], n = tiles_of(a, g);
      if (lane == 0) {
        if (clamp_ctx(c, a) != c) set_err(a.err, IR_DEVERR_CONTEXT_LEN);
        ri->start = 0;
        ri->end = n;
        ri->b_first = g;
        ri->p_first = 0;
      }
      if (n == 0 && !a.keep_empty) {
        T* o = reinterpret_cast<T*>(a.out) + g * a.out_stride +
               static_cast<int64_t>(kv0) * a.n_rep * D;
        for (int i = lane; i < HG * a.n_rep * D; i += 32) o[i] = DT<T>::from_f(0.f);
      }
      __syncwarp();
    }
  } else if (a.B <= 32 * kEach) {
    if (warp == 0) {
      int64_t sum = 0;
      int n[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int sb = lane * kEach + i;
        n[i] = sb < a.B ? a.context_lens[sb] : 0;
      }
      bool bad = false;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int c = clamp_ctx(n[i], a);
        bad = bad || c != n[i];
        n[i] = (c + kTile - 1) / kTile;
        sum += n[i];
      }
      if (bad) set_err(a.err, IR_DEVERR_CONTEXT_LEN);
      int64_t incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(kFull, incl, o);
        if (lane >= o) incl += y;
      }
      const int64_t total = __shfl_sync(kFull, incl, 31);
      const int G = shares_used(total, a.G);
      const int64_t from = g < G ? share_start(g, total, G) : total;
      const int64_t to = g < G ? share_start(g + 1, total, G) : total;
      int64_t p = incl - sum;
      if (sum > 0 && p <= from && from < incl) {  // one lane, where the share is not empty
        int i = 0;
#pragma unroll
        for (int k = 0; k < kEach - 1; ++k)
          if (i == k && from >= p + n[k]) p += n[k], ++i;
        ri->b_first = lane * kEach + i;
        ri->p_first = p;
      }
      if (lane == 0) ri->start = from, ri->end = to;
      __syncwarp();
    } else if (!a.keep_empty) {
      for (int sb = (warp - 1) * a.G + g; sb < a.B; sb += kConsumers * a.G) {
        if (clamp_ctx(a.context_lens[sb], a) != 0) continue;
        T* o = reinterpret_cast<T*>(a.out) + sb * a.out_stride +
               static_cast<int64_t>(kv0) * a.n_rep * D;
        for (int i = lane; i < HG * a.n_rep * D; i += 32) o[i] = DT<T>::from_f(0.f);
      }
    }
  } else {
    find_share<kThreads, T>(a, g, kv0, HG, ri, sm_scan);
  }

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    // Lane i resolves tile t + i: its sequence, block and scales. Tiles of one
    // aligned group of W lanes and one segment are an item, led by their
    // first lane; then, item by item, the lanes of an item issue their own
    // copies and store their own scales, so that little is left to do between
    // a stage falling free and its copies.
    const int64_t start = ri->start, end = ri->end;
    int b = 0, nb = 0;
    int64_t pb = 0;
    if (start < end) {
      b = ri->b_first;
      pb = ri->p_first;
      nb = tiles_of(a, b);
    }
    int seg = -1;  // segments started before this batch, less one
    uint32_t slot = 0, par = 1;
    bool abort = false;
    const float* kscale = a.k_scale + kv0;
    const float* vscale = a.v_scale + kv0;
    for (int64_t t = start; t < end && !abort; t += 32) {
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
      int nvalid = 0, id0 = 0, id1 = -1, row0 = 0;
      bool ok = false, seg_start = false;
      if (active) {
        const int tok0 = j * kTile;
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
      }
      const bool whole = (lp >= start) && (lp + ln <= end);
      // scales [block][side][head] of this tile (in flight until they are stored)
      float sc[NB * 2 * HG];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int64_t id = i == 0 ? id0 : id1;
#pragma unroll
        for (int h = 0; h < HG; ++h) {
          sc[(2 * i) * HG + h] = ok && id >= 0 ? kscale[id * a.Hkv + h] : 0.f;
          sc[(2 * i + 1) * HG + h] = ok && id >= 0 ? vscale[id * a.Hkv + h] : 0.f;
        }
      }
      const unsigned starts = __ballot_sync(kFull, active && seg_start);
      const unsigned oks = __ballot_sync(kFull, ok);
      const unsigned lead = __ballot_sync(kFull, active && (seg_start || lane % W == 0));
      const unsigned upto = lane == 31 ? kFull : (2u << lane) - 1u;
      const unsigned mine = lead & upto;  // leaders up to this lane: the last is its own
      const int leader = active ? 31 - __clz(mine) : -1;
      const unsigned after = lead & ~upto;
      const int nact = (end - t) < 32 ? static_cast<int>(end - t) : 32;
      // for leaders: tiles of the item, valid tokens, bytes and flags
      const int n = (after ? __ffs(after) - 1 : nact) - lane;
      const int last = __shfl_sync(kFull, nvalid, (lane + n - 1) & 31);
      const unsigned issued = (oks >> lane) & ((1u << (n > 0 ? n : 0)) - 1u);
      const int kseg = seg + __popc(starts & upto);
      uint32_t bytes = __popc(issued) * static_cast<uint32_t>(L::kTileBytes);
      if (R == 8 && last <= 8 && n > 0 && ((issued >> (n - 1)) & 1u)) bytes -= 2u * L::kBox;
      const ItemQ8 it{lb, g, (n - 1) * kTile + last,
                      static_cast<int>(issued) | (seg_start ? kSegStart : 0) |
                          (whole ? kWhole : 0) | ((kseg & 1) ? kQBuf1 : 0)};
      const uint32_t qrows = static_cast<uint32_t>(HG * a.n_rep * D * 2);

      for (unsigned left = lead; left != 0; left &= left - 1) {
        const int k = __ffs(left) - 1;
        bool good = mbar_wait_bounded(&empty[slot], par);
        if (q_bulk && ((starts >> k) & 1u)) {
          const int sg = __shfl_sync(kFull, kseg, k);
          if (sg >= 2) good = good && mbar_wait_bounded(&qfree[sg & 1], ((sg >> 1) + 1) & 1);
        }
        if (!__all_sync(kFull, good)) {
          if (lane == 0) set_err(a.err, IR_DEVERR_TIMEOUT);
          abort = true;
          break;
        }
        if (leader == k) {
          uint8_t* td = smem + slot * L::kStage + (lane - k) * L::kTileBytes;
          if (ok) {
            tma_load_3d(td, &tmk, &full[slot], 0, row0, kv0);
            tma_load_3d(td + L::kSide, &tmv, &full[slot], 0, row0, kv0);
            if (R == 8 && id1 >= 0) {
              tma_load_3d(td + L::kBox, &tmk, &full[slot], 0, id1 * a.bs, kv0);
              tma_load_3d(td + L::kSide + L::kBox, &tmv, &full[slot], 0, id1 * a.bs, kv0);
            }
          }
          if (lane == k) {
            desc[slot] = it;
            if (q_bulk && seg_start)
              bulk_load(smem + L::off_q + (kseg & 1) * q_buf,
                        reinterpret_cast<const T*>(a.q) + lb * a.q_stride +
                            static_cast<int64_t>(kv0 * a.n_rep) * D,
                        qrows, &full[slot]);
          }
          float* so = scales + slot * L::kScales + (lane - k) * (NB * 2 * HG);
#pragma unroll
          for (int i = 0; i < NB * 2 * HG; ++i) so[i] = sc[i];
        }
        __syncwarp();
        if (lane == k) mbar_arrive_expect_tx(&full[slot], bytes + (q_bulk && seg_start ? qrows : 0u));
        if (++slot == NS) {
          slot = 0;
          par ^= 1u;
        }
      }
      seg += __popc(starts);
      b = __shfl_sync(kFull, lb, nact - 1);
      pb = __shfl_sync(kFull, lp, nact - 1);
      nb = __shfl_sync(kFull, ln, nact - 1);
    }
    if (!abort) {
      const bool good = mbar_wait_bounded(&empty[slot], par);
      if (lane == 0) {
        if (good) {
          desc[slot] = ItemQ8{0, 0, 0, kEnd};
          mbar_arrive(&full[slot]);
        } else {
          set_err(a.err, IR_DEVERR_TIMEOUT);
        }
      }
      abort = !__all_sync(kFull, good);
    }
    // (given up: the copies under way still need this shared memory)
    if (abort)
      for (int i = 0; i < NS; ++i)
        mbar_wait_bounded(&full[i], static_cast<uint32_t>(i) < slot ? par ^ 1u : par);
    return;
  }

  // -------------------------------------------------------------- consumers
  const int cw = warp - 1;
  const int row = cw / WT, part = cw % WT;  // the state this warp shares, its place there
  const int first = row * WT;               // place of the row's first warp
  const int head = SETS ? row / 2 : row, set = SETS ? row % 2 : 0;
  const int kvh = kv0 + head;
  const int n0 = SETS ? set * 8 : 0;             // first query head of the set
  const int nq = min(8, a.n_rep - n0);           // query heads of the set
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

  float acc[KS][4];
  float m[2], l[2], qinv[2] = {0.f, 0.f};
  uint32_t qf[KS][2];
  auto reset = [&]() {
#pragma unroll
    for (int i = 0; i < KS; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  };
  reset();
#pragma unroll
  for (int i = 0; i < KS; ++i) qf[i][0] = qf[i][1] = 0u;
  int seg_b = -1, seg_unit = 0;
  bool seg_whole = false, have_seg = false;
  uint32_t flushes = 0;

  // Combine the WT states of the finished segment and write its rows: the
  // output (whole sequences) or a normalised fp32 piece. In each step the
  // upper half of the remaining warps hands its (m, l) and O to the lower half
  // and is done; the buffer it writes is the one it last read (in the first
  // step the reader's own, once its readers of the last segment are through).
  auto flush = [&]() {
    uint64_t* bar = hbar + first;
    float2* ml = reinterpret_cast<float2*>(smem + L::off_ml) + first * 8 + qd;
    // 16-byte pieces of a lane's D / 8 columns, rotated by its rows against bank conflicts
    float* parts = reinterpret_cast<float*>(smem + L::off_part) + row * (WT / 2) * L::kPart +
                   qd * D + pc * (D / 8);
    auto piece = [&](int i) { return ((i / 2) ^ (qq & (D / 32 - 1))) * 4; };
    const uint32_t par = flushes & 1u;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      l[j] += __shfl_xor_sync(kFull, l[j], 4);
      l[j] += __shfl_xor_sync(kFull, l[j], 8);
      l[j] += __shfl_xor_sync(kFull, l[j], 16);
    }
    int mine = part >= WT / 2 ? part - WT / 2 : part;  // buffer of this warp
    if (WT > 1 && part >= WT / 2 && flushes > 0 &&
        !__all_sync(kFull, mbar_wait_bounded(&bar[0], par ^ 1u)))
      return false;
    ++flushes;
    for (int h = WT / 2; h > 0; h >>= 1) {
      if (part >= h) {
        float* o = parts + mine * L::kPart;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (grp == 0) ml[part * 8 + j] = make_float2(m[j], l[j]);
#pragma unroll
          for (int i = 0; i < KS; i += 2)
            *reinterpret_cast<float4*>(o + j * D + piece(i)) =
                make_float4(acc[i][j], acc[i][j + 2], acc[i + 1][j], acc[i + 1][j + 2]);
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bar[part]);
          if (part < WT / 2) mbar_arrive(&bar[0]);  // (a reader of the steps before)
        }
        break;
      }
      if (!__all_sync(kFull, mbar_wait_bounded(&bar[part + h], par))) return false;
      mine = h == WT / 2 ? part : mine + h;
      const float* o = parts + mine * L::kPart;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 other = ml[(part + h) * 8 + j];
        const float M = fmaxf(m[j], other.x);
        const float use = M == -INFINITY ? 0.f : M;
        const float f = ex2(m[j] - use), e = ex2(other.x - use);
        l[j] = l[j] * f + other.y * e;
        m[j] = M;
#pragma unroll
        for (int i = 0; i < KS; i += 2) {
          const float4 x = *reinterpret_cast<const float4*>(o + j * D + piece(i));
          acc[i][j] = acc[i][j] * f + x.x * e;
          acc[i][j + 2] = acc[i][j + 2] * f + x.y * e;
          acc[i + 1][j] = acc[i + 1][j] * f + x.z * e;
          acc[i + 1][j + 2] = acc[i + 1][j + 2] * f + x.w * e;
        }
      }
    }
    if (part == 0) {
      if (WT > 1) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar[0]);
      }
      const int64_t pslot = static_cast<int64_t>(kvh) * a.ws_slots + seg_unit + seg_b;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = n0 + qd + j;
        // nothing attended: zero (a NaN sum is not nothing)
        const float f = l[j] == 0.f ? 0.f : 1.f / l[j];
        if (qd + j >= nq) continue;
        if (seg_whole) {
          T* dst = reinterpret_cast<T*>(a.out) + seg_b * a.out_stride +
                   static_cast<int64_t>(kvh * a.n_rep + n) * D + pc * (D / 8);
#pragma unroll
          for (int i = 0; i < KS; i += 4)
            *reinterpret_cast<uint4*>(dst + 2 * i) =
                make_uint4(pack2<T>(acc[i][j] * f, acc[i][j + 2] * f),
                           pack2<T>(acc[i + 1][j] * f, acc[i + 1][j + 2] * f),
                           pack2<T>(acc[i + 2][j] * f, acc[i + 2][j + 2] * f),
                           pack2<T>(acc[i + 3][j] * f, acc[i + 3][j + 2] * f));
        } else {
          float* dst = a.ws_o + (pslot * a.n_rep + n) * D + pc * (D / 8);
#pragma unroll
          for (int i = 0; i < KS; i += 2)
            *reinterpret_cast<float4*>(dst + 2 * i) =
                make_float4(acc[i][j] * f, acc[i][j + 2] * f, acc[i + 1][j] * f,
                            acc[i + 1][j + 2] * f);
          if (grp == 0)
            a.ws_lse[pslot * a.n_rep + n] =
                l[j] == 0.f ? -INFINITY : m[j] + log2f(l[j]) - kPShift;
        }
      }
    }
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
      const int hr = n0 + grp;  // query head of the group
      float v[D / 4];
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < D / 4; ++e) v[e] = 0.f;
      if (hr < a.n_rep) {
        if (q_bulk) {
          const uint4* src = reinterpret_cast<const uint4*>(
              smem + L::off_q + buf * q_buf + (head * a.n_rep + hr) * D * 2);
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
        qf[i][0] = pack2<__half>(v[o] * up, v[o + 1] * up);
        qf[i][1] = pack2<__half>(v[o + 2] * up, v[o + 3] * up);
      }
      const float inv = down * a.scale_log2;
      qinv[0] = __shfl_sync(kFull, inv, qd * 4);
      qinv[1] = __shfl_sync(kFull, inv, (qd + 1) * 4);
      if (q_bulk) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&qfree[buf]);
      }
    }
    // this warp's tiles of the item (short items are spread over the warps)
    int nv[kPair];
#pragma unroll
    for (int u = 0; u < kPair; ++u) {
      const int w = u * WT + part;
      nv[u] = ((it.flags >> w) & 1) ? max(0, min(kTile, it.ntok - w * kTile)) : 0;
    }
    if (nv[0] | nv[kPair - 1]) {
      const uint32_t base = smem_u32(smem + slot * L::kStage + part * L::kTileBytes) +
                            head * L::kRegion;
      constexpr int kApart = WT * L::kTileBytes;  // from one of its tiles to the next
      const float* sc = scales + slot * L::kScales + part * (NB * 2 * HG) + head;
      // scales of each tile's first and second 8 tokens (0 where there are none)
      float ks[kPair][2], vs[kPair][2];
#pragma unroll
      for (int u = 0; u < kPair; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bool any = nv[u] > (NB == 2 ? 8 * i : 0);
          const float* q = sc + (u * WT * NB + (NB == 2 ? i : 0)) * 2 * HG;
          ks[u][i] = any ? q[0] : 0.f;
          vs[u][i] = any ? q[HG] : 0.f;
        }

      // S^T of both tiles; two accumulators each halve the dependent chain
      float s[kPair][4], t[kPair][4];
#pragma unroll
      for (int u = 0; u < kPair; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u][i] = t[u][i] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
#pragma unroll
        for (int u = 0; u < kPair; ++u) {
          const uint32_t kb = base + u * kApart + koff[c];
          const uint4 x = lds128(kb), y = lds128(kb + kHalf);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t a0, a1, a2, a3;
            decode4_h<C>(xs[e], a0, a2);
            decode4_h<C>(ys[e], a1, a3);
            mma_16816<__half>((e & 1) ? t[u] : s[u], a0, a1, a2, a3, qf[c * 4 + e][0],
                              qf[c * 4 + e][1]);
          }
        }

      // V codes: their reads overlap the softmax
      constexpr int VW = D / 32;  // words per lane and token
      uint32_t vw[kPair][4][VW];
#pragma unroll
      for (int u = 0; u < kPair; ++u) {
        const uint32_t vb0 = base + u * kApart + L::kSide;
        const uint32_t at[4] = {vb0 + va, vb0 + vb, vb0 + kHalf + va, vb0 + kHalf + vb};
        const int tk[4] = {ta, tb, ta + 8, tb + 8};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (D == 128) {
            const uint4 x = lds128(at[i]);
            vw[u][i][0] = x.x, vw[u][i][1] = x.y, vw[u][i][2] = x.z, vw[u][i][3] = x.w;
          } else {
            const uint2 x = lds64(at[i]);
            vw[u][i][0] = x.x, vw[u][i][1] = x.y;
          }
        }
        if (nv[u] < kTile) {
          // rows past the context may hold NaN codes, and 0 * NaN is NaN
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (tk[i] >= nv[u]) {
#pragma unroll
              for (int e = 0; e < VW; ++e) vw[u][i][e] = 0u;
            }
        }
      }

      // scores in log2 units (registers of s), [tile][half * 2 + head column]
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int u = 0; u < kPair; ++u) {
        const bool v0 = tg < nv[u], v1 = tg + 8 < nv[u];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          s[u][j] = v0 ? (s[u][j] + t[u][j]) * (qinv[j] * ks[u][0]) : -INFINITY;
          s[u][j + 2] = v1 ? (s[u][j + 2] + t[u][j + 2]) * (qinv[j] * ks[u][1]) : -INFINITY;
          mx[j] = max3(mx[j], s[u][j], s[u][j + 2]);
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mx[j] = fmaxf(mx[j], __shfl_xor_sync(kFull, mx[j], 4));
        mx[j] = fmaxf(mx[j], __shfl_xor_sync(kFull, mx[j], 8));
        mx[j] = fmaxf(mx[j], __shfl_xor_sync(kFull, mx[j], 16));
      }
      const bool up0 = mx[0] > m[0] + kSlack, up1 = mx[1] > m[1] + kSlack;
      if (__any_sync(kFull, up0 || up1)) {
        const float a0 = up0 ? ex2(m[0] - mx[0]) : 1.f, a1 = up1 ? ex2(m[1] - mx[1]) : 1.f;
        if (up0) m[0] = mx[0];
        if (up1) m[1] = mx[1];
        l[0] *= a0;
        l[1] *= a1;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          acc[i][0] *= a0;
          acc[i][1] *= a1;
          acc[i][2] *= a0;
          acc[i][3] *= a1;
        }
      }
      const float r0 = kPShift - (m[0] == -INFINITY ? 0.f : m[0]);
      const float r1 = kPShift - (m[1] == -INFINITY ? 0.f : m[1]);
      uint32_t pb[kPair][2];
#pragma unroll
      for (int u = 0; u < kPair; ++u) {
        const float p0 = ex2(s[u][0] + r0), p1 = ex2(s[u][1] + r1);
        const float p2 = ex2(s[u][2] + r0), p3 = ex2(s[u][3] + r1);
        l[0] += p0 + p2;
        l[1] += p1 + p3;
        pb[u][0] = movmatrix_trans(pack2<__half>(p0, p1));
        pb[u][1] = movmatrix_trans(pack2<__half>(p2, p3));
      }

      // O^T += vs * (V^T . P^T)
      auto add = [&](float* o, const float* x, float v) {
        const unsigned long long v2 = f2pack(v, v);
        const float2 y = f2unpack(fma2(v2, f2pack(x[0], x[1]), f2pack(o[0], o[1])));
        const float2 z = f2unpack(fma2(v2, f2pack(x[2], x[3]), f2pack(o[2], o[3])));
        o[0] = y.x, o[1] = y.y, o[2] = z.x, o[3] = z.y;
      };
#pragma unroll
      for (int e = 0; e < VW; ++e)
#pragma unroll
        for (int u = 0; u < kPair; ++u) {
          uint32_t a0[2], a1[2], a2[2], a3[2];
          decode4_h<C>(__byte_perm(vw[u][0][e], vw[u][1][e], 0x5140), a0[0], a1[0]);
          decode4_h<C>(__byte_perm(vw[u][0][e], vw[u][1][e], 0x7362), a0[1], a1[1]);
          decode4_h<C>(__byte_perm(vw[u][2][e], vw[u][3][e], 0x5140), a2[0], a3[0]);
          decode4_h<C>(__byte_perm(vw[u][2][e], vw[u][3][e], 0x7362), a2[1], a3[1]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float x[4] = {0.f, 0.f, 0.f, 0.f};
            mma_16816<__half>(x, a0[i], a1[i], a2[i], a3[i], pb[u][0], NB == 1 ? pb[u][1] : 0u);
            add(acc[2 * e + i], x, vs[u][0]);
            if (NB == 2) {  // two blocks: their products apart
              float y[4] = {0.f, 0.f, 0.f, 0.f};
              mma_16816<__half>(y, a0[i], a1[i], a2[i], a3[i], 0u, pb[u][1]);
              add(acc[2 * e + i], y, vs[u][1]);
            }
          }
        }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[slot]);
  }
}

// ---------------------------------------------------------------- merge
//
// The pieces of a row (query head of a sequence) that several CTAs hold,
// combined by W warps, every warp loading up to U pieces at once and lane i
// columns 4 i .. 4 i + 3. The grid should be resident while the decode CTAs
// still run, so that nothing but the pieces' round trip remains after them:
// beside a decode CTA an SM has a quarter of its registers and 2-4 KB of
// shared memory left. Hence rows of one group in one CTA without shared
// memory where a row has few pieces (W = 1), and four warps a row otherwise.
// Which pieces a row has follows from the context lengths, summed by every
// warp before the wait for batches of up to 256 (else the decode grid's prefix).
template <typename T, int W, int U>
__global__ void __launch_bounds__(W == 1 ? 256 : 32 * W) merge_q8_kernel(const DecodeArgs a) {
  launch_dependents();
  constexpr int kSide = W > 1 ? W : 1;
  __shared__ float4 s_acc[W > 1 ? W : 1][W > 1 ? 32 : 1];
  __shared__ float2 s_ms[kSide];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x, kvh = blockIdx.y;
  const bool early = a.B <= 256;
  int64_t total = 0, pb = 0, nb = 0;
  int glo = 0, parts = 0;
  auto units = [&]() {
    if (nb > 0) piece_range(pb, nb, total, shares_used(total, a.G), &glo, &parts);
  };
  if (early) {
    for (int i = lane; i < a.B; i += 32) {
      const int64_t t = tiles_of(a, i);
      total += t;
      if (i < b) pb += t;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      total += __shfl_xor_sync(kFull, total, o);
      pb += __shfl_xor_sync(kFull, pb, o);
    }
    nb = tiles_of(a, b);
    units();
  }
  wait_prerequisites();
  if (!early) {
    pb = a.ws_prefix[b];
    nb = a.ws_prefix[b + 1] - pb;
    total = a.ws_prefix[a.B];
    units();
  }
  if (nb <= 0 || parts == 1) return;  // empty, or written whole by its CTA
  const bool active = lane * 4 < a.D;
  // W = 1: a warp per row of the group in turns; else the CTA's row is in z
  const int step = W == 1 ? blockDim.x >> 5 : a.n_rep;
  for (int n = W == 1 ? warp : blockIdx.z; n < a.n_rep; n += step) {
    const int64_t base = static_cast<int64_t>(kvh) * a.ws_slots + glo + b;
    const float* lse = a.ws_lse + base * a.n_rep + n;
    const float* o = a.ws_o + (base * a.n_rep + n) * a.D + lane * 4;
    const int64_t ostride = static_cast<int64_t>(a.n_rep) * a.D;
    float M = -INFINITY, S = 0.f;
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = W == 1 ? 0 : warp; i0 < parts; i0 += W * U) {
      float li[U];
      float4 oi[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * W;
        li[u] = -INFINITY;
        oi[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < parts) {
          li[u] = __ldcg(lse + static_cast<int64_t>(i) * a.n_rep);
          if (active) oi[u] = __ldcg(reinterpret_cast<const float4*>(o + i * ostride));
        }
      }
      float top = M;
#pragma unroll
      for (int u = 0; u < U; ++u) top = fmaxf(top, li[u]);
      const float use = top == -INFINITY ? 0.f : top;
      const float c = ex2(M - use);
      S *= c;
      r.x *= c, r.y *= c, r.z *= c, r.w *= c;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float w = ex2(li[u] - use);  // (0 for a piece with nothing attended)
        S += w;
        r.x += w * oi[u].x, r.y += w * oi[u].y, r.z += w * oi[u].z, r.w += w * oi[u].w;
      }
      M = top;
    }
    if (W > 1) {
      s_acc[warp][lane] = r;
      if (lane == 0) s_ms[warp] = make_float2(M, S);
      __syncthreads();
      if (warp != 0) return;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, s_ms[w].x);
      const float use = top == -INFINITY ? 0.f : top;
      S = 0.f;
      r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float c = ex2(s_ms[w].x - use);
        const float4 x = s_acc[w][lane];
        S += c * s_ms[w].y;
        r.x += c * x.x, r.y += c * x.y, r.z += c * x.z, r.w += c * x.w;
      }
    }
    if (active) {
      const float f = S == 0.f ? 0.f : 1.f / S;  // (a NaN sum is not nothing)
      T* dst = reinterpret_cast<T*>(a.out) + b * a.out_stride +
               static_cast<int64_t>(kvh * a.n_rep + n) * a.D + lane * 4;
      *reinterpret_cast<uint2*>(dst) =
          make_uint2(pack2<T>(r.x * f, r.y * f), pack2<T>(r.z * f, r.w * f));
    }
  }
}

template <typename T>
int launch_merge_q8(const DecodeArgs& a, cudaStream_t s) {
  // a sequence of average length spans about G / B shares (+ 1)
  const int pieces = a.G / (a.B > 0 ? a.B : 1) + 1;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = s;
  if (pieces <= 8) {
    cfg.gridDim = dim3(a.B, a.Hkv);
    cfg.blockDim = dim3(32 * (a.n_rep < 8 ? a.n_rep : 8));
    return static_cast<int>(cudaLaunchKernelEx(&cfg, merge_q8_kernel<T, 1, 4>, a));
  }
  cfg.gridDim = dim3(a.B, a.Hkv, a.n_rep);
  cfg.blockDim = dim3(32 * 4);
  return static_cast<int>(cudaLaunchKernelEx(&cfg, merge_q8_kernel<T, 4, 10>, a));
}

// ---------------------------------------------------------------- dispatch

struct CallQ8 {
  const CUtensorMap *tmk, *tmv;
  const DecodeArgs* a;
  int q_bulk;
  cudaStream_t s;
};

template <typename T, typename C, int D, int HG, int R, bool SETS>
int run_q8(const CallQ8* call) {
  constexpr int NS = stages_q8<D, HG, R, SETS>();
  using L = LayoutQ8<D, HG, R, NS, SETS>;
  static_assert(L::kAlloc <= 227 * 1024 && NS >= 3, "shared memory budget");
  auto kern = decode_q8_kernel<T, C, D, HG, R, SETS, NS>;
  // the shared-memory limit is set on a device's first launch (a bit each; those
  // beyond 63 every time), and once more if a launch fails, since a device
  // reset takes it back
  static std::atomic<uint64_t> known{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
  bool fresh = !(known.load(std::memory_order_acquire) & bit);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(call->a->Hkv / HG, call->a->G);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::bytes(call->a->n_rep);
  cfg.stream = call->s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  for (;;) {
    if (fresh) {
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kAlloc);
      if (e != cudaSuccess) return static_cast<int>(e);
      known.fetch_or(bit, std::memory_order_release);
    }
    e = cudaLaunchKernelEx(&cfg, kern, *call->tmk, *call->tmv, *call->a, call->q_bulk);
    if (e == cudaSuccess || fresh) return static_cast<int>(e);
    cudaGetLastError();  // (not sticky: the launch was refused)
    fresh = true;
  }
}

template <typename T, typename C, int D, int HG, bool SETS>
int by_rows(const CallQ8* c) {
  return c->a->bs == 8 ? run_q8<T, C, D, HG, 8, SETS>(c) : run_q8<T, C, D, HG, 16, SETS>(c);
}
template <typename T, typename C, int D>
int by_heads(const CallQ8* c) {
  const int hg = c->a->per_seq ? c->a->per_seq : q8_head_group(c->a->Hkv, c->a->n_rep);
  if (c->a->n_rep <= 8) {
    switch (hg) {
      case 1: return by_rows<T, C, D, 1, false>(c);
      case 2: return by_rows<T, C, D, 2, false>(c);
      case 4: return by_rows<T, C, D, 4, false>(c);
      default: return by_rows<T, C, D, 8, false>(c);
    }
  }
  switch (hg) {
    case 1: return by_rows<T, C, D, 1, true>(c);
    case 2: return by_rows<T, C, D, 2, true>(c);
    default: return by_rows<T, C, D, 4, true>(c);
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

// Heads of a CTA that takes a whole sequence, 0: shares. Short contexts do without
// the share search and the merge, with as few heads a CTA as leave all CTAs in one
// wave. Against shares, 28 / 4 heads of 128 (contexts of the tables' width): 1 x 201
// 6.6 us and 8.2, 64 x 201 7.7 and 13.8, 128 x 512 16.3 and 22.6, 64 x 1024 15.9 and
// 20.9; but 1 x 1024 12.0 and 9.4, 128 x 1024 with 8 / 8 ragged 45 and 33.
int q8_seq_heads(int batch, int num_kv_heads, int n_rep, int64_t max_ctx, int sms) {
  for (int hg : {1, 2, 4, 8})
    if (num_kv_heads % hg == 0 && (hg < 8 || n_rep <= 8) &&
        static_cast<int64_t>(batch) * (num_kv_heads / hg) <= sms)
      return max_ctx <= 512 || (max_ctx <= 1024 && batch >= 16 && hg <= 2) ? hg : 0;
  return 0;
}

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
  const bool bf16 = dtype == IR_DTYPE_BF16;
  const int e = bf16 ? by_code<__nv_bfloat16>(fmt, &call) : by_code<__half>(fmt, &call);
  if (e || a.per_seq) return e;
  return bf16 ? launch_merge_q8<__nv_bfloat16>(a, stream) : launch_merge_q8<__half>(a, stream);
}

}  // namespace irb
