// sqa_scaled.cu -- attention over a block-scaled e4m3 cache, and the attention weight of
// every cached token, on the 5th-generation tensor cores.
//
// Orientation.  The tokens are the M side of both products: S^T = K Q^T puts token t of a
// 128-token block (8 pages) on TMEM lane t and the query rows on columns, and O^T += V^T P^T
// puts the head dimension on lanes and the rows on columns.  A softmax thread then owns one
// token: its page's two scales are two scalars of the thread (a factor of every score of the
// lane, and of every probability it writes), a token's attention weight is a sum over the
// thread's own registers, and the M = 128 side is full whatever q_len is (with rows on M, a
// q_len of 4 fills 16 of 128 lanes).
//
// Precision.  The tensor core reads the e4m3 K and V as they are (kind::f8f6f4 wants 8-bit
// operands on both sides).  Q and P enter as sums of e4m3 numbers, x = x0 + x1 / 32 +
// x2 / 1024 .., each the e4m3 rounding of what the parts before it left (4 significant bits a
// part).  The parts are extra columns of the N side (free: an M = 128 product of few columns
// is bound by reading A) with their own fp32 accumulators, joined at read-out, so that a
// low part has its own exponent range.  Two parts hold a bf16 query exactly (8 bits), three an fp16
// query (11 bits).  Q is first scaled by the power of two that brings the largest finite
// magnitude of the head's rows into [128, 256); there the smallest part resolves 2^-15 (bf16) or 2^-20
// (fp16), which is 2^-22 or 2^-27 of that magnitude, and rows far below it lose bits under that.
// P has four parts, the last one 2^20 times too large: P is held to 2^-13 of it, below 2^-11 to
// 2^-24, of which no more than 2^-4 of P, and lost only below 2^-30.  That matters for a row
// that one token dominates, where the many others lie 2^-19 and further below it and still add up:
// with three parts they left the numerator (a tail of 0.26 came out as 0.17 or 0).  Such a row's
// base is chosen so that they lie higher (kRest).  The fourth part fits in the columns that 16 rows
// leave unused.
//
// Softmax.  A row keeps a base; a score with its value scale, y = c ks (q . k) + log2 vs, enters as
// P = 2^(y - base), and the denominator sums P / vs.  The value scale is thus inside the running
// maximum, and P keeps its e4m3 range whatever the pages' value scales are.  Bases are set from the
// first block to its maxima + 1 (less where one token dominates) and raised when some y exceeds its base by more than 8 (one
// barrier with an or-reduction a block finds that out; then every row whose block maximum passed
// its old one is raised, and l and O are rescaled).  Raising costs a block as much again, and on
// random data with 1% of fourfold tokens it came in every second to fifth block with 3 to 6 bits
// of slack: hence 9, which the low parts of P leave room for.  Masked tokens and tokens behind
// the sequence have y = -inf by selection, so NaN in their K does not matter; V rows behind the
// sequence are zeroed in shared memory, and a NaN in the V of a draft token is zeroed and
// remembered, as only the rows that see the token get it.
//
// Weights.  w_t = sum over the rows of 2^(c ks (q . k) - lse): the same score product, summed over the
// thread's columns and added to the token's score.  16-bit caches use kind::f16 and Q as it is.
//
// Streams.  A unit is a (block, group of 16 rows); each of W softmax warpgroups takes every W-th unit: of
// one group always, with its own bases and O, and the streams of a group are joined at the
// end of a piece.  Two for up to 32 rows, four beyond (96 registers a thread): with one
// warpgroup a block of 64 rows took 13.7k cycles, with two of 32 rows 6.9k, with four of 16
// 3.8k; at 32 rows two beat four (237 against 248 us at 16 x 8 x 32768), and 16 rows a group beat 32
// (237 / 241 us, fp16 243 / 290, for want of registers).  Two groups of a block share a product
// (GP = 2, one read of K and V for both: 4 x 16 x 65536 230 -> 195 us).
//
// What bounds it.  q_len 1-4 run at 5.2-5.7 TB/s (q_len 2, 16 x 32768: 190 us for 1.07 GB), near what
// the loads alone reach (5.8 TB/s at q_len 4 with P, the scores and the value products left out).  Above it
// is the softmax threads' work, more than any one stage: with three parts of P, at q_len 8, of 245 us,
// leaving out P saved 28, the scores 18, the value products 38, all three 45; at q_len 16 (4 x 65536, before
// GP = 2), of 238 us, 29, 25, 60 and 79.  The fourth part took q_len 8 from 241 to 261 us and q_len 16 (1 x 262144)
// from 194 to 219, where the SM now issues 2.6 instructions a cycle.
//
// Warps: 0 .. 4 W - 1 softmax (one token a thread), then one each for score products, value
// products, TMA and page scales.  Work is cut into CTA ranges by sqa_schedule.cuh; pieces of a split
// segment are merged by sqa_scaled_merge_kernel.
//
// Pipelines (mbarriers; every wait bounded):
//   full / empty [tiles]     producer -> issuers; K and V tiles (16 KB) alternate in one ring,
//                            each released by the commit of the product that read it
//   s_full / s_empty [NS]    score issuer (commit) -> softmax -> score issuer
//   p_full / p_done [2 LANES]  softmax -> value issuer (commit) -> softmax, two P buffers a lane
//   q_ready [2]              softmax (Q of a piece, one piece ahead) -> score issuer
//   m_full / m_empty [8]     page scales of a block -> softmax
#include <atomic>

#include "small_q_attention.h"
#include "sqa_internal.h"
#include "sqa_merge_row.cuh"
#include "sqa_ptx.cuh"
#include "sqa_scaled.cuh"
#include "sqa_schedule.cuh"

namespace sqa {
namespace {

constexpr int kBlockPages = 8;
constexpr int kBlock = kBlockPages * kPageSize;  // 128 tokens: the M side
constexpr int kTileBytes = kBlock * 128;         // K or V of a block (e4m3), or one half of 16-bit K
constexpr int kMetaSlots = 8;
constexpr int kPParts = 4;                       // e4m3 parts of a probability: P = p0 + p1 / 32 + p2 / 2^10 + p3 / 2^20
constexpr float kLastPart = 1024.f;              // of p3 against p2
constexpr float kRaise = 8.f, kHead = -1.f;      // raise a base that a score exceeds by 2^8, to 2 times the maximum
// A row that one token dominates keeps the rest at 2^-12 or more, as far as the largest P may go for it: 2^7 in a
// stream's first block, 2^4 later, where the next larger token would have the base raised again.
constexpr float kRest = 12.f, kTopFirst = 7.f, kTopLater = 4.f;
constexpr float kLn2f = 0.6931471805599453f;
// 2^-60: smaller value scales count as this.  With none over 2^30, the documented limit, y - base underflows (under
// -126) only for tokens of 2^-35 and less of the largest probability; over 2^60 it would from 2^-5 on.
constexpr float kMinValueScale = 8.673617379884035e-19f;

// PARTS: e4m3 parts of Q, 2 or 3; 0 = 16-bit cache (weights only).
// ROWS: query rows of a group, G groups, W streams (softmax warpgroups).
template <int PARTS_, int ROWS_, int G_, int W_, bool ATTEND_>
struct Shape {
  static constexpr int PARTS = PARTS_, ROWS = ROWS_, G = G_, W = W_;
  static constexpr bool ATTEND = ATTEND_, F8 = PARTS_ > 0;
  static constexpr int SOFTMAX = W * 128, THREADS = SOFTMAX + 128;
  static constexpr int COLS = (F8 ? PARTS : 1) * ROWS;
  static constexpr int N = (COLS + 15) / 16 * 16;             // score columns of a group (N of the product)
  static constexpr int GP = ATTEND && G > 1 ? 2 : 1;          // groups that one product takes: A is read once for both
  static constexpr int UNITS = G / GP;                        // products of a block, each for GP streams
  static constexpr int SN = GP * N;
  static constexpr int STRIDE = SN <= 16 ? 16 : SN <= 32 ? 32 : SN <= 64 ? 64 : 128;  // TMEM columns of a score slot
  static constexpr int PROW = 64;                             // bytes of a token's P in a group: four parts of 16 rows
  static constexpr int PPITCH = GP * PROW;                    // and of its operand row
  static constexpr int PBYTES = kBlock * PPITCH;
  static constexpr int LANES = W / GP;                        // streams of products
  static constexpr int OCOLS = ATTEND ? W * PROW : 0;         // O^T of the streams
  static constexpr int SLOTS_FIT = (512 - OCOLS) / STRIDE;
  static constexpr int NS = SLOTS_FIT < 8 ? SLOTS_FIT : 8;
  static constexpr int Q_GROUP = F8 ? N * 128 : 2 * N * 128;  // bytes of one group's Q operand
  static constexpr int Q_BYTES = G * Q_GROUP;
  static constexpr int TILES = ATTEND || !F8 ? 2 : 1;         // 16 KB tiles of a block (K and V, or K's two halves)
  static constexpr int Q_STEPS = (G * ROWS * 8 + SOFTMAX - 1) / SOFTMAX;
  static_assert(!ATTEND || (kPParts * ROWS <= PROW && W % G == 0), "columns");
  // A slot belongs to one warpgroup (or pair): only then does a wait see no phase but the next one.
  static_assert(NS % (ATTEND ? LANES : W * G) == 0, "slots");
  static_assert(SN <= 128 && NS >= 2 && NS <= 8 && W <= 4 && G * ROWS <= 64, "columns");
};

struct ScaledTcParams {
  SplitKvParams s;  // schedule, tables, outputs (s.out: 16-bit rows; s.out_o: fp32 rows; s.out_lse: optional)
  const float* k_scales;
  const float* v_scales;
  long long scale_stride;
  const float* lse;  // weights
  float* scores;
};

// Shared memory of a CTA: everything of a fixed size first (so that its addresses are one register
// plus constants), then the ring of tiles.
template <class S>
struct Smem {
  static constexpr int kMaxTiles = 16;
  static constexpr int P = 0;                                           // two P buffers for each lane of products
  static constexpr int Q = P + (S::ATTEND ? S::LANES * 2 * S::PBYTES : 0);    // two Q slots
  static constexpr int META = Q + 2 * S::Q_BYTES;                       // [kMetaSlots][8]: ks, log2 vs, 1 / vs, page id (bits)
  static constexpr int BASE = META + kMetaSlots * kBlockPages * 16;     // [W][ROWS]: a stream's bases (weights: -lse of all rows)
  static constexpr int DELTA = BASE + 64 * 4;                           // [W][ROWS]: raises; the epilogue's factors of O
  static constexpr int WRED = DELTA + 64 * 4;                           // [4 W][ROWS]: per-warp maxima, then sums
  static constexpr int NAN_FROM = WRED + 256 * 4;                       // [W][128]
  static constexpr int CQ = NAN_FROM + S::W * 128 * 4;              // [2]: log2-domain score factor of a Q slot
  static constexpr int QTOP = CQ + 16;                                  // [16]
  static constexpr int SCH = QTOP + 64;
  static constexpr int TMEM = SCH + 64;
  static constexpr int FULL = TMEM + 16;  // barriers
  static constexpr int EMPTY = FULL + kMaxTiles * 8;
  static constexpr int S_FULL = EMPTY + kMaxTiles * 8;
  static constexpr int S_EMPTY = S_FULL + 8 * 8;
  static constexpr int P_FULL = S_EMPTY + 8 * 8;
  static constexpr int P_DONE = P_FULL + 2 * S::W * 8;
  static constexpr int Q_READY = P_DONE + 2 * S::W * 8;
  static constexpr int M_FULL = Q_READY + 2 * 8;
  static constexpr int M_EMPTY = M_FULL + kMetaSlots * 8;
  static constexpr int DONE = M_EMPTY + kMetaSlots * 8;
  static constexpr int RING = (DONE + 8 + 1023) / 1024 * 1024;
  static_assert((!S::ATTEND || S::W * S::ROWS <= 64) && sizeof(Schedule) <= 64 && META % 1024 == 0 && FULL % 8 == 0, "layout");

  uint8_t* at;  // 1024-byte aligned, in shared memory

  __device__ __forceinline__ uint8_t* ring(int tile) const { return at + RING + tile * kTileBytes; }
  // the buffer of a lane's v-th product, and the index of its barriers
  __device__ __forceinline__ static int pi(int lane, int v) { return 2 * lane + (v & 1); }
  __device__ __forceinline__ uint8_t* p(int lane, int v) const { return at + P + pi(lane, v) * S::PBYTES; }
  __device__ __forceinline__ uint8_t* q(int slot) const { return at + Q + slot * S::Q_BYTES; }
  __device__ __forceinline__ float4* meta(int slot) const { return reinterpret_cast<float4*>(at + META) + slot * kBlockPages; }
  __device__ __forceinline__ float* base(int stream) const { return reinterpret_cast<float*>(at + BASE) + stream * S::ROWS; }
  __device__ __forceinline__ float* delta(int stream) const { return reinterpret_cast<float*>(at + DELTA) + stream * S::ROWS; }
  __device__ __forceinline__ float* wred(int warp) const { return reinterpret_cast<float*>(at + WRED) + warp * S::ROWS; }
  __device__ __forceinline__ int* nan_from() const { return reinterpret_cast<int*>(at + NAN_FROM); }
  __device__ __forceinline__ float* cq() const { return reinterpret_cast<float*>(at + CQ); }
  __device__ __forceinline__ unsigned int* qtop() const { return reinterpret_cast<unsigned int*>(at + QTOP); }
  __device__ __forceinline__ Schedule* sch() const { return reinterpret_cast<Schedule*>(at + SCH); }
  __device__ __forceinline__ uint32_t* tmem() const { return reinterpret_cast<uint32_t*>(at + TMEM); }
  __device__ __forceinline__ uint32_t bar(int group, int i = 0) const { return smem_u32(at) + group + i * 8; }
};

// The pieces of a CTA's range: f(walk, first unit, pages) for each, in order.
template <class F>
__device__ __forceinline__ void for_pieces(const SplitKvParams& p, const Schedule& sch, F f) {
  SegWalk w = first_segment(p, sch);
  int unit = sch.start;
  while (unit < sch.end) {
    const int seg_end = w.seg_start + w.pages;
    const int n = min(sch.end, seg_end) - unit;
    f(w, unit, n);
    unit += n;
    if (unit >= seg_end) next_segment(p, w);
    else w.pg += n;
  }
}

__device__ __forceinline__ int blocks_of(int pages) { return (pages + kBlockPages - 1) / kBlockPages; }

// As for_pieces, by a whole warp, with the piece's page ids: f(walk, c0, n, id) for each chunk of 32
// pages from page c0 of the piece on, lane l holding the id of page c0 + l.  The ids are read one
// chunk ahead, across pieces too.
template <class F>
__device__ __forceinline__ void for_page_chunks(const SplitKvParams& p, const Schedule& sch, F f) {
  const int lane = threadIdx.x & 31;
  SegWalk w = first_segment(p, sch);
  int unit = sch.start;
  auto first_ids = [&](const SegWalk& x, int u) {
    const int n = min(sch.end, x.seg_start + x.pages) - u;
    return lane < n ? __ldg(p.block_tables + (size_t)x.b * p.max_pages + x.pg + lane) : 0;
  };
  int ids = unit < sch.end ? first_ids(w, unit) : 0;
  while (unit < sch.end) {
    const int n = min(sch.end, w.seg_start + w.pages) - unit;
    const int32_t* row = p.block_tables + (size_t)w.b * p.max_pages + w.pg;
    const int next = unit + n;
    SegWalk wn = w;
    if (next < sch.end) next_segment(p, wn);  // a piece ends at its segment's end or the range's
    for (int c0 = 0; c0 < n; c0 += 32) {
      int ahead = 0;
      if (c0 + 32 < n) ahead = c0 + 32 + lane < n ? __ldg(row + c0 + 32 + lane) : 0;
      else if (next < sch.end) ahead = first_ids(wn, next);
      f(w, c0, n, ids);
      ids = ahead;
    }
    unit = next;
    w = wn;
  }
}

// ------------------------------------------------------------------ producer (whole warp)
template <class S>
__device__ void produce(const ScaledTcParams& p, const Schedule& sch, const CUtensorMap* tm_k, const CUtensorMap* tm_v,
                        const Smem<S>& sm, int tiles, volatile int* abort) {
  const uint64_t policy = l2_policy_evict_first();
  int slot = 0, issued = 0;
  uint32_t phase = 0;
  unsigned int bad = 0;
  for_page_chunks(p.s, sch, [&](const SegWalk& w, int c0, int n, int id) {
    // NHD map: (dim, head, token, page); HND map: (dim, token, head, page)
    const int c1 = p.s.hnd ? 0 : w.h, c2 = p.s.hnd ? w.h : 0;
    const int cnt = min(32, n - c0);
    for (int jb = 0; jb < cnt; jb += kBlockPages) {
      const int np = min(kBlockPages, cnt - jb);
      int pages[kBlockPages];
#pragma unroll
      for (int j = 0; j < kBlockPages; ++j) {
        pages[j] = __shfl_sync(0xffffffffu, id, min(jb + j, 31));
        if (j < np && (pages[j] < 0 || pages[j] >= p.s.num_pages)) {
          bad = 1;
          pages[j] = 0;
        }
      }
#pragma unroll
      for (int tile = 0; tile < S::TILES; ++tile) {  // K then V; or the two 64-dim halves of 16-bit K
        bool ok = mbar_wait_bounded(sm.bar(Smem<S>::EMPTY, slot), phase ^ 1u, abort, p.s.status);
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (ok) {
          if (elect_one()) {
            const uint32_t f = sm.bar(Smem<S>::FULL, slot);
            mbar_arrive_expect_tx(f, np * 2048);
            const uint32_t dst = smem_u32(sm.ring(slot));
            const CUtensorMap* map = (S::F8 && tile == 1) ? tm_v : tm_k;
            const int c = S::F8 ? 0 : tile * 64;
            for (int j = 0; j < np; ++j) tma_load_4d(dst + j * 2048, map, f, c, c1, c2, pages[j], policy);
          }
          __syncwarp();
          ++issued;
        }
        if (++slot == tiles) {
          slot = 0;
          phase ^= 1u;
        }
      }
    }
  });
  const int lane = threadIdx.x & 31;
  if (__any_sync(0xffffffffu, bad) && lane == 0) atomicOr(p.s.status, 8u);  // SQA_DEV_BAD_PAGE
  if (lane == 0 && *abort) {  // only an abort can leave loads in flight
    for (int k = 0; k < min(issued, tiles); ++k) {
      const int last = k + tiles * ((issued - 1 - k) / tiles);
      if (!mbar_drain(sm.bar(Smem<S>::FULL, k), (uint32_t)(last / tiles) & 1u, 100000000ull))
        atomicOr(p.s.status, 1u);
    }
  }
}

// ------------------------------------------------------------------ page scales (whole warp)
// The scales (and, for the weights, the id) of every page of a block into a meta slot.
template <class S>
__device__ void page_meta(const ScaledTcParams& p, const Schedule& sch, const Smem<S>& sm, volatile int* abort) {
  const int lane = threadIdx.x & 31;
  int blk = 0;
  for_page_chunks(p.s, sch, [&](const SegWalk& w, int c0, int n, int id) {
    const bool in = c0 + lane < n;
    const bool good = id >= 0 && id < p.s.num_pages;
    float4 m = make_float4(S::F8 ? 0.f : 1.f, 0.f, 1.f, __int_as_float(in && good ? id : -1));
    if (S::F8 && in) {
      const size_t at = (size_t)(good ? id : 0) * p.scale_stride + w.h;
      m.x = __ldcg(p.k_scales + at);  // through L2: the append before may have run beside this grid's start
      if (S::ATTEND) {
        const float vs = fmaxf(__ldcg(p.v_scales + at), kMinValueScale);
        m.y = log2f(vs);
        m.z = 1.f / vs;
      }
    }
    const int cnt = min(32, n - c0);
    for (int jb = 0; jb < cnt; jb += kBlockPages, ++blk) {
      const int e = blk % kMetaSlots;
      if (blk >= kMetaSlots)
        mbar_wait_bounded(sm.bar(Smem<S>::M_EMPTY, e), (uint32_t)(blk / kMetaSlots - 1) & 1u, abort, p.s.status);
      if (lane >= jb && lane < jb + kBlockPages) sm.meta(e)[lane - jb] = m;
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.bar(Smem<S>::M_FULL, e));
    }
  });
}

// ------------------------------------------------------------------ product issuers (whole warps, one elected lane)
__device__ __forceinline__ void tc_mma_ss_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <class S>
__device__ __forceinline__ void drain_products(const ScaledTcParams& p, const Smem<S>& sm) {
  if (elect_one()) tc_commit(sm.bar(Smem<S>::DONE));
  __syncwarp();
  if (!mbar_drain(sm.bar(Smem<S>::DONE), 0u, 2000000000ull) && (threadIdx.x & 31) == 0)
    atomicOr(p.s.status, 1u);
}

// A running position in the ring of tiles.
struct RingPos {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int tiles) {
    if (++slot == tiles) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// S^T of product u, (block, GP groups), into score slot u % NS.
template <class S, bool BF>
__device__ void issue_scores(const ScaledTcParams& p, const Schedule& sch, const Smem<S>& sm, uint32_t tmem, int tiles,
                             volatile int* abort) {
  constexpr uint32_t kIdesc = mma_idesc_f16(128, S::SN, false, false, BF && !S::F8);  // format 0: e4m3 / fp16
  int u = 0, pc = 0;
  RingPos at;
  for_pieces(p.s, sch, [&](const SegWalk&, int, int n) {
    mbar_wait_bounded(sm.bar(Smem<S>::Q_READY, (pc & 1)), (uint32_t)(pc >> 1) & 1u, abort, p.s.status);
    const uint32_t q = smem_u32(sm.q(pc & 1));
    const int nblk = blocks_of(n);
    for (int k = 0; k < nblk; ++k) {
      const int k0 = at.slot;  // K's tile (its first half)
      mbar_wait_bounded(sm.bar(Smem<S>::FULL, at.slot), at.phase, abort, p.s.status);
      at.next(tiles);
      const int k1 = at.slot;
      if (!S::F8) mbar_wait_bounded(sm.bar(Smem<S>::FULL, at.slot), at.phase, abort, p.s.status);
      if (S::TILES == 2) at.next(tiles);  // K's second half, or V
#pragma unroll 1
      for (int g = 0; g < S::UNITS; ++g, ++u) {
        if (u >= S::NS)
          mbar_wait_bounded(sm.bar(Smem<S>::S_EMPTY, u % S::NS), (uint32_t)(u / S::NS - 1) & 1u, abort, p.s.status);
        __syncwarp();
        tc_fence_after();
        if (elect_one()) {
          const uint32_t d = tmem + S::OCOLS + (u % S::NS) * S::STRIDE;
          const uint32_t qg = q + g * S::GP * S::Q_GROUP;
          const uint32_t kt = smem_u32(sm.ring(k0));
          if constexpr (S::F8) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)  // 32 dims (32 B) a step
              tc_mma_ss_f8(d, smem_desc_sw128(kt + kk * 32, 16, 1024), smem_desc_sw128(qg + kk * 32, 16, 1024), kIdesc,
                           kk > 0 ? 1u : 0u);
          } else {
            const uint32_t kt1 = smem_u32(sm.ring(k1));
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)  // 16 dims (32 B) a step, four to a half
              tc_mma_ss(d, smem_desc_sw128((kk < 4 ? kt : kt1) + (kk & 3) * 32, 16, 1024),
                        smem_desc_sw128(qg + (kk >> 2) * (S::N * 128) + (kk & 3) * 32, 16, 1024), kIdesc, kk > 0 ? 1u : 0u);
          }
          tc_commit(sm.bar(Smem<S>::S_FULL, u % S::NS));
          if (g == S::UNITS - 1) {  // the block's K may be overwritten
            tc_commit(sm.bar(Smem<S>::EMPTY, k0));
            if (!S::F8) tc_commit(sm.bar(Smem<S>::EMPTY, k1));
          }
        }
        __syncwarp();
      }
    }
    ++pc;
  });
  drain_products(p, sm);
}

// Descriptor of P, MN-major: one atom of PPITCH rows (bytes) x 8 tokens, swizzled over its row.
template <class S>
__device__ __forceinline__ uint64_t desc_p(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)((S::PBYTES >> 4) & 0x3FFFu) << 16;     // between atoms along the rows: there is one
  d |= (uint64_t)((8 * S::PPITCH >> 4) & 0x3FFFu) << 32;  // between groups of 8 tokens
  d |= (uint64_t)1 << 46;                                // version
  d |= (uint64_t)(S::PPITCH == 128 ? 2 : 4) << 61;       // SWIZZLE_128B or SWIZZLE_64B
  return d;
}

// O^T of the streams of lane u % LANES += V^T P^T of product u, once their P is in the lane's buffer.
template <class S>
__device__ void issue_values(const ScaledTcParams& p, const Schedule& sch, const Smem<S>& sm, uint32_t tmem, int tiles,
                             volatile int* abort) {
  constexpr uint32_t kIdesc = mma_idesc_f16(128, S::PPITCH, true, true, false);
  int u = 0;
  RingPos at;
  for_pieces(p.s, sch, [&](const SegWalk&, int, int n) {
    const int nblk = blocks_of(n);
    for (int k = 0; k < nblk; ++k) {
      at.next(tiles);  // over K
      const int np = min(kBlockPages, n - k * kBlockPages);
      mbar_wait_bounded(sm.bar(Smem<S>::FULL, at.slot), at.phase, abort, p.s.status);
#pragma unroll 1
      for (int g = 0; g < S::UNITS; ++g, ++u) {
        const int st = u % S::LANES, v = u / S::LANES;
        mbar_wait_bounded(sm.bar(Smem<S>::P_FULL, sm.pi(st, v)), (uint32_t)(v >> 1) & 1u, abort, p.s.status);
        __syncwarp();
        tc_fence_after();
        if (elect_one()) {
          const uint32_t vt = smem_u32(sm.ring(at.slot));
          const uint32_t pb = smem_u32(sm.p(st, v));
          const int steps = (np + 1) / 2;  // 32 tokens a step; the softmax zeroed an absent page's V
          // a stream's first product of a piece overwrites O
          for (int kk = 0; kk < steps; ++kk)
            tc_mma_ss_f8(tmem + st * S::PPITCH, smem_desc_sw128(vt + kk * 4096, kTileBytes, 1024), desc_p<S>(pb + kk * 32 * S::PPITCH),
                         kIdesc, (k >= S::W / S::G || kk > 0) ? 1u : 0u);
          tc_commit(sm.bar(Smem<S>::P_DONE, sm.pi(st, v)));
          if (g == S::UNITS - 1) tc_commit(sm.bar(Smem<S>::EMPTY, at.slot));
        }
        __syncwarp();
      }
      at.next(tiles);
    }
  });
  drain_products(p, sm);
}

// ------------------------------------------------------------------ softmax warps (128 threads)
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}

// Barrier of a softmax warpgroup; true when `v` is for any of its threads.
__device__ __forceinline__ bool group_any(int stream, bool v) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, 128, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((int)v), "r"(1 + stream)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void group_sync(int stream) { named_bar_sync(1 + stream, 128); }
template <class S>
__device__ __forceinline__ void softmax_sync() {
  named_bar_sync(1 + S::W, S::SOFTMAX);
}

// The four e4m3 parts of two probabilities below 2^8.  Differences of a number and its rounding
// are exact; 32 times the first one is taken in fp32 and rounded to fp16 (2^-16 of P, and 2^-30).  The last part
// saturates above P = 16, where the first three hold P to 2^-13.
__device__ __forceinline__ void split_p(float x0, float x1, uint32_t (&out)[kPParts]) {
  out[0] = e4m3x2_of_floats(x0, x1);
  const float2 f = __half22float2(__hmul2(half2_of_e4m3x2(out[0]), __floats2half2_rn(-32.f, -32.f)));
  const __half2 h = __floats2half2_rn(fmaf(x0, 32.f, f.x), fmaf(x1, 32.f, f.y));
  out[1] = e4m3x2_of_half2(h);
  const __half2 g = __hmul2(__hsub2(h, half2_of_e4m3x2(out[1])), __floats2half2_rn(32.f, 32.f));
  out[2] = e4m3x2_of_half2(g);
  out[3] = e4m3x2_of_half2(__hmul2(__hsub2(g, half2_of_e4m3x2(out[2])), __floats2half2_rn(kLastPart, kLastPart)));
}

// PARTS e4m3 parts of four numbers, exact differences: x = part 0 + part 1 / 32 + part 2 / 1024.
template <int PARTS>
__device__ __forceinline__ void split_q(float (&x)[4], uint32_t (&out)[3]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const uint32_t a = pack_e4m3x2(x[0], x[1]), b = pack_e4m3x2(x[2], x[3]);
    out[i] = a | (b << 16);
    if (i + 1 < PARTS) {
      const float2 fa = unpack_e4m3x2(a), fb = unpack_e4m3x2(b);
      x[0] = (x[0] - fa.x) * 32.f;
      x[1] = (x[1] - fa.y) * 32.f;
      x[2] = (x[2] - fb.x) * 32.f;
      x[3] = (x[3] - fb.y) * 32.f;
    }
  }
}

// Q of (b, h) as the N operand of the score product: row r of part i is operand row i * ROWS + r of its
// group (128 B, 128-byte swizzle).  All softmax threads, eight to a row, 16 dims each.
template <class S>
struct QItem {
  uint4 x[S::Q_STEPS][2];
  uint32_t top[S::Q_STEPS];  // the row's largest magnitude, as bits (above every finite one for infinity and NaN)
};

// The thread's part of Q into registers, and the warp's largest finite magnitude into qtop.
template <class S, bool BF>
__device__ __forceinline__ void load_q(const ScaledTcParams& p, const Smem<S>& sm, int b, int h, QItem<S>& q) {
  uint32_t most = 0;
#pragma unroll
  for (int st = 0; st < S::Q_STEPS; ++st) {
    const int it = st * S::SOFTMAX + threadIdx.x, r = it >> 3, c = it & 7;
    q.x[st][0] = q.x[st][1] = make_uint4(0u, 0u, 0u, 0u);
    if (r < kGroup * p.s.q_len) {
      const __half* src =
          p.s.q + ((size_t)(b * p.s.q_len + (r >> 2)) * p.s.hq + h * kGroup + (r & 3)) * kHeadDim + c * 16;
      q.x[st][0] = __ldg(reinterpret_cast<const uint4*>(src));
      q.x[st][1] = __ldg(reinterpret_cast<const uint4*>(src) + 1);
    }
  }
  if constexpr (S::F8) {
#pragma unroll
    for (int st = 0; st < S::Q_STEPS; ++st) {
      const uint32_t w[8] = {q.x[st][0].x, q.x[st][0].y, q.x[st][0].z, q.x[st][0].w,
                             q.x[st][1].x, q.x[st][1].y, q.x[st][1].z, q.x[st][1].w};
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 a = unpack2<BF>(w[i]);
        top = max(top, max(__float_as_uint(a.x) & 0x7fffffffu, __float_as_uint(a.y) & 0x7fffffffu));
      }
#pragma unroll
      for (int off = 1; off < 8; off <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
      q.top[st] = top;
      if (top < 0x7f800000u) most = max(most, top);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if ((threadIdx.x & 31) == 0) sm.qtop()[threadIdx.x >> 5] = most;
  }
}

// After a barrier of the softmax threads: the thread's part of Q into slot `qs`.
template <class S, bool BF>
__device__ __forceinline__ void write_q(const ScaledTcParams& p, const Smem<S>& sm, const QItem<S>& q, int qs) {
  uint32_t most = 0;
  if constexpr (S::F8) {
#pragma unroll
    for (int i = 0; i < S::SOFTMAX / 32; ++i) most = max(most, sm.qtop()[i]);
  }
  // 2^e brings the largest magnitude into [128, 256)
  const int e = most > 0 ? max(-110, min(110, 134 - (int)(most >> 23))) : 0;
  if (threadIdx.x == 0) sm.cq()[qs] = p.s.scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
  for (int st = 0; st < S::Q_STEPS; ++st) {
    const int it = st * S::SOFTMAX + threadIdx.x, r = it >> 3, c = it & 7;
    if (r >= S::G * S::ROWS) break;
    const int rr = r % S::ROWS;
    uint8_t* const dst = sm.q(qs) + (r / S::ROWS) * S::Q_GROUP;
    if constexpr (!S::F8) {  // 32 bytes of half c / 4: chunks 2 (c % 4) and the next
      uint8_t* const row = dst + (c >> 2) * (S::N * 128) + (rr >> 3) * 1024 + (rr & 7) * 128;
      const int c0 = (c & 3) * 2;
      *reinterpret_cast<uint4*>(row + ((c0 ^ (rr & 7)) << 4)) = q.x[st][0];
      *reinterpret_cast<uint4*>(row + (((c0 + 1) ^ (rr & 7)) << 4)) = q.x[st][1];
    } else {
      const float sc = __uint_as_float((uint32_t)(127 + e) << 23);
      const uint32_t w[8] = {q.x[st][0].x, q.x[st][0].y, q.x[st][0].z, q.x[st][0].w,
                             q.x[st][1].x, q.x[st][1].y, q.x[st][1].z, q.x[st][1].w};
      uint32_t part[3][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = unpack2<BF>(w[2 * i]), d = unpack2<BF>(w[2 * i + 1]);
        float y[4] = {a.x * sc, a.y * sc, d.x * sc, d.y * sc};
        uint32_t o[3];
        split_q<S::PARTS>(y, o);
#pragma unroll
        for (int k = 0; k < S::PARTS; ++k)  // a row with an infinity or NaN is NaN
          part[k][i] = q.top[st] < 0x7f800000u ? o[k] : 0x7f7f7f7fu;
      }
#pragma unroll
      for (int k = 0; k < S::PARTS; ++k) {
        const int n = k * S::ROWS + rr;
        *reinterpret_cast<uint4*>(dst + (n >> 3) * 1024 + (n & 7) * 128 + ((c ^ (n & 7)) << 4)) =
            make_uint4(part[k][0], part[k][1], part[k][2], part[k][3]);
      }
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(sm.bar(Smem<S>::Q_READY, qs));
}

// Rows [c, c + 8) of a score slot, its parts joined.
template <class S>
__device__ __forceinline__ void read_scores(uint32_t slot, int c, float (&s)[8]) {
  constexpr int kParts = S::F8 ? S::PARTS : 1;
  uint32_t raw[kParts][8];
#pragma unroll
  for (int i = 0; i < kParts; ++i) tmem_ld(slot + i * S::ROWS + c, raw[i]);
  tmem_wait_ld();
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    float x = __uint_as_float(raw[kParts - 1][r]);
#pragma unroll
    for (int i = kParts - 2; i >= 0; --i) x = fmaf(x, 1.f / 32.f, __uint_as_float(raw[i][r]));
    s[r] = x;
  }
}

// Each row's sum or maximum over the warp's lanes: lane l gets row l / (32 / ROWS).  Halves the rows a
// lane holds at each step (ROWS + 1 shuffles instead of 5 ROWS).
template <int ROWS, bool MAX>
__device__ __forceinline__ float reduce_rows(const float (&in)[ROWS]) {
  auto join = [](float a, float b) { return MAX ? fmaxf(a, b) : a + b; };
  const int lane = threadIdx.x & 31;
  float v[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) v[i] = in[i];
  int n = ROWS;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    if (n > 1) {
      n /= 2;
      const bool upper = lane & off;
#pragma unroll
      for (int i = 0; i < ROWS / 2; ++i) {
        if (i < n) {
          const float mine = upper ? v[i + n] : v[i], other = upper ? v[i] : v[i + n];
          v[i] = join(mine, __shfl_xor_sync(0xffffffffu, other, off));
        }
      }
    } else {
      v[0] = join(v[0], __shfl_xor_sync(0xffffffffu, v[0], off));
    }
  }
  return v[0];
}

// What the softmax threads know of a piece.
struct Piece {
  int len, first;  // tokens held; tokens that draft row 0 sees (its limit: mask - q_len + 1)
  int fresh;       // the step's own tokens, the last q_len of the whole sequence, start here
};

__device__ __forceinline__ Piece piece_of(const SplitKvParams& p, const SegWalk& w) {
  const int raw = __ldg(p.seq_lens + w.b);
  const int whole = p.mask_lens ? __ldg(p.mask_lens + w.b) : raw;
  return Piece{min(raw, w.pages * kPageSize), whole - p.q_len + 1, whole - p.q_len};
}

// t = y - base of a unit's rows, and their largest; `release` is called once the scores are in registers.
// MASK: the block holds tokens that some row does not see (late: see attend).
template <class S, bool MASK, class F>
__device__ __forceinline__ float unit_scores(uint32_t slot, const float* base, float kc, float lv, int late, int row0,
                                             float (&t)[S::ROWS], F release) {
  uint32_t raw[S::ROWS / 8][S::PARTS][8];
#pragma unroll
  for (int c = 0; c < S::ROWS / 8; ++c)
#pragma unroll
    for (int i = 0; i < S::PARTS; ++i) tmem_ld(slot + i * S::ROWS + c * 8, raw[c][i]);
  tmem_wait_ld();
  release();
  float over = -INFINITY;
#pragma unroll
  for (int r = 0; r < S::ROWS; r += 4) {
    const float4 b4 = *reinterpret_cast<const float4*>(base + r);
    const float bb[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = (r + i) / 8, e = (r + i) % 8;
      float s = __uint_as_float(raw[c][S::PARTS - 1][e]);
#pragma unroll
      for (int j = S::PARTS - 2; j >= 0; --j) s = fmaf(s, 1.f / 32.f, __uint_as_float(raw[c][j][e]));
      float x = fmaf(s, kc, lv - bb[i]);
      if (MASK && late >= (row0 + r + i) >> 2) x = -INFINITY;
      t[r + i] = x;
      over = fmaxf(over, x);
    }
  }
  return over;
}

// The scales of block bk's page of this thread's token.
template <class S>
__device__ __forceinline__ float4 read_meta(const ScaledTcParams& p, const Smem<S>& sm, int bk, volatile int* abort) {
  const int e = bk % kMetaSlots;
  mbar_wait_bounded(sm.bar(Smem<S>::M_FULL, e), (uint32_t)(bk / kMetaSlots) & 1u, abort, p.s.status);
  const float4 m = sm.meta(e)[(threadIdx.x & 127) >> 4];
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(sm.bar(Smem<S>::M_EMPTY, e));
  return m;
}

template <class S, bool BF>
__device__ void attend(const ScaledTcParams& p, const Schedule& sch, const Smem<S>& sm, uint32_t tmem, int tiles,
                       volatile int* abort) {
  constexpr int ROWS = S::ROWS, G = S::G, W = S::W;
  constexpr int kStep = W / G;  // blocks from unit to unit of a stream
  const int stream = threadIdx.x >> 7;
  const int tid = threadIdx.x & 127, warp = tid >> 5, lane = tid & 31;  // tid: token of a block, dimension of O
  const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
  const int rows = kGroup * p.s.q_len;
  const int group = stream % G;  // the stream's rows: row0 .. row0 + ROWS - 1
  const int row0 = group * ROWS;
  const int plane = stream / S::GP;  // its lane of products
  float* const base = sm.base(stream);
  float* const delta = sm.delta(stream);
  float* const wred = sm.wred(stream * 4);
  if (p.s.seg_split == 1 && sch.start >= sch.end) {  // no merge follows: a sequence without tokens
    const int b = (int)blockIdx.x / p.s.hkv, h = (int)blockIdx.x - b * p.s.hkv;
    for (int r = stream; r < rows; r += W) {
      const size_t out_row = (size_t)(b * p.s.q_len + (r >> 2)) * p.s.hq + h * kGroup + (r & 3);
      if (p.s.out_o) p.s.out_o[out_row * kHeadDim + tid] = 0.f;
      else reinterpret_cast<uint16_t*>(p.s.out)[out_row * kHeadDim + tid] = 0;
      if (p.s.out_lse && tid == 0) p.s.out_lse[out_row] = -INFINITY;
    }
  }
  int blk = 0, pc = 0;
  for_pieces(p.s, sch, [&](const SegWalk& w, int unit, int n) {
    const int seg = w.b * p.s.hkv + w.h;
    const int seg_end = w.seg_start + w.pages;
    const bool whole = unit == w.seg_start && seg_end <= sch.end;
    const Piece piece = piece_of(p.s, w);
    if (pc == 0) {
      QItem<S> q;
      load_q<S, BF>(p, sm, w.b, w.h, q);
      if (tid < ROWS) base[tid] = 0.f;
      softmax_sync<S>();
      write_q<S, BF>(p, sm, q, 0);
      softmax_sync<S>();
    }
    const float cq = sm.cq()[pc & 1];
    float l[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) l[r] = 0.f;
    int nan_from = 0x7fffffff;  // first draft token whose V is NaN in dimension tid

    const int nblk = blocks_of(n);
    const int k0 = (stream / G - blk) & (kStep - 1);  // the stream's first block of the piece
    float4 meta = make_float4(0.f, 0.f, 0.f, 0.f);
    if (k0 < nblk) meta = read_meta(p, sm, blk + k0, abort);
    for (int k = k0; k < nblk; k += kStep) {
      const int bk = blk + k;
      const int u = bk * S::UNITS + group / S::GP;  // product
      const int v = u / S::LANES;                   // the stream's own count
      const int np = min(kBlockPages, n - k * kBlockPages);
      const int tok0 = (w.pg + k * kBlockPages) * kPageSize;
      const int tok = tok0 + tid;
      const bool masked = np < kBlockPages || tok0 + kBlock > piece.first || tok0 + kBlock > piece.len;
      // draft qi sees the token iff late < qi (every draft when negative)
      const int late = (tid < np * kPageSize && tok < piece.len) ? tok - piece.first : 0x7fffffff;

      if (masked && group == 0) {
        // V rows behind the sequence and of absent pages: zero (they may hold NaN); draft tokens'
        // NaN: zero, and remembered by the dimension's thread.  (The block's first group does it: its
        // product comes first.)
        const int t1 = bk * 2 + 1;  // V's tile
        // The tile's last occupant is tiles / 2 > kStep blocks back: once the lane's last product is done,
        // and with it every product before, its barrier is in no earlier phase than the one waited for.
        if (v >= 1)
          mbar_wait_bounded(sm.bar(Smem<S>::P_DONE, sm.pi(plane, v - 1)), (uint32_t)((v - 1) >> 1) & 1u, abort, p.s.status);
        mbar_wait_bounded(sm.bar(Smem<S>::FULL, t1 % tiles), (uint32_t)(t1 / tiles) & 1u, abort, p.s.status);
        uint8_t* const vt = sm.ring(t1 % tiles);
        const int held = min(np * kPageSize, max(piece.len - tok0, 0));
        const int read = (np + 1) / 2 * 32;  // rows that the product reads
        for (int t = max(0, piece.first - tok0); t < held; ++t) {
          uint8_t* const at = vt + t * 128 + (((tid >> 4) ^ (t & 7)) << 4) + (tid & 15);
          if ((*at & 0x7f) == 0x7f) {
            nan_from = min(nan_from, tok0 + t);
            *at = 0;
          }
        }
        for (int c = held * 8 + tid; c < read * 8; c += 128)
          *reinterpret_cast<uint4*>(vt + c * 16) = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
      }

      mbar_wait_bounded(sm.bar(Smem<S>::S_FULL, u % S::NS), (uint32_t)(u / S::NS) & 1u, abort, p.s.status);
      tc_fence_after();
      const uint32_t slot = lanes + S::OCOLS + (u % S::NS) * S::STRIDE + (group % S::GP) * S::N;
      float t[ROWS];
      const float kc = meta.x * cq;
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sm.bar(Smem<S>::S_EMPTY, u % S::NS));
      };
      const float over = masked ? unit_scores<S, true>(slot, base, kc, meta.y, late, row0, t, release)
                                : unit_scores<S, false>(slot, base, kc, meta.y, late, row0, t, release);
      const float inv_vs = meta.z;
      if (k + kStep < nblk) meta = read_meta(p, sm, bk + kStep, abort);  // off the next unit's path
      const bool first = k == k0;
      const bool raise = group_any(stream, over > kRaise) || first;  // rare after a piece's first blocks
      if (raise) {
        const float m = reduce_rows<ROWS, true>(t);
        if (lane % (32 / ROWS) == 0) wred[warp * ROWS + lane / (32 / ROWS)] = m;
        group_sync(stream);
        if (tid < ROWS) {
          const float w0 = wred[tid], w1 = wred[ROWS + tid], w2 = wred[2 * ROWS + tid], w3 = wred[3 * ROWS + tid];
          const float m4 = fmaxf(fmaxf(w0, w1), fmaxf(w2, w3));
          const float rest = fminf(fminf(w0, w1), fminf(w2, w3));  // a token that dominates is in one of the warps
          float d = 0.f;
          if (m4 > kHead || (first && m4 != -INFINITY)) {
            d = fmaxf(m4 - (first ? kTopFirst : kTopLater), fminf(m4 - kHead, rest + kRest));
            if (!first) d = fmaxf(d, 0.f);
          }
          delta[tid] = d;
          base[tid] += d;
        }
        group_sync(stream);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) t[r] -= delta[r];
      }
      if (raise && !first) {  // O stands still once the stream's last product is done
        mbar_wait_bounded(sm.bar(Smem<S>::P_DONE, sm.pi(plane, v - 1)), (uint32_t)((v - 1) >> 1) & 1u, abort, p.s.status);
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < ROWS; c += 8) {
          float a[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            a[r] = ex2(-delta[c + r]);
            l[c + r] *= a[r];
          }
#pragma unroll
          for (int i = 0; i < kPParts; ++i) {
            uint32_t o[8];
            tmem_ld(lanes + stream * S::PROW + i * ROWS + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int r = 0; r < 8; ++r) o[r] = __float_as_uint(__uint_as_float(o[r]) * a[r]);
            tmem_st8(lanes + stream * S::PROW + i * ROWS + c, o);
          }
        }
        tmem_wait_st();
      }
      // P: token tid's operand row of PPITCH bytes, in the group's 64 part i of row r in byte
      // i * ROWS + r; 16-byte chunks swizzled by the token
      // (its buffer is free once the product before the last is done)
      if (v >= 2) mbar_wait_bounded(sm.bar(Smem<S>::P_DONE, sm.pi(plane, v)), (uint32_t)((v >> 1) - 1) & 1u, abort, p.s.status);
      uint8_t* const prow = sm.p(plane, v) + tid * S::PPITCH;
      const int swizzle = S::PPITCH == 128 ? tid & 7 : (tid >> 1) & 3;
      constexpr int kHalf = ROWS < 16 ? ROWS : 16;  // rows of a 16-byte chunk
#pragma unroll
      for (int c = 0; c < ROWS; c += kHalf) {
        uint32_t part[kPParts][kHalf / 4];
#pragma unroll
        for (int r = 0; r < kHalf; r += 4) {
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[i] = ex2(t[c + r + i]);
            l[c + r + i] = fmaf(x[i], inv_vs, l[c + r + i]);
          }
          uint32_t lo[kPParts], hi[kPParts];
          split_p(x[0], x[1], lo);
          split_p(x[2], x[3], hi);
#pragma unroll
          for (int i = 0; i < kPParts; ++i) part[i][r / 4] = lo[i] | (hi[i] << 16);
        }
#pragma unroll
        for (int i = 0; i < kPParts; ++i) {
          const int byte = (group % S::GP) * S::PROW + i * ROWS + c;
          uint8_t* const at = prow + (((byte >> 4) ^ swizzle) << 4) + (byte & 15);
          if constexpr (kHalf == 16)
            *reinterpret_cast<uint4*>(at) = make_uint4(part[i][0], part[i][1], part[i][2], part[i][3]);
          else
            *reinterpret_cast<uint2*>(at) = make_uint2(part[i][0], part[i][1]);
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.bar(Smem<S>::P_FULL, sm.pi(plane, v)));
    }

    // ---- epilogue: denominators and factors, then each dimension's thread joins its rows' parts
    const bool more = seg_end < sch.end;  // another piece follows: its Q, for the score products
    QItem<S> q;
    if (more) {
      SegWalk nw = w;
      next_segment(p.s, nw);
      load_q<S, BF>(p, sm, nw.b, nw.h, q);
    }
    const float total = reduce_rows<ROWS, false>(l);
    if (lane % (32 / ROWS) == 0) wred[warp * ROWS + lane / (32 / ROWS)] = total;
    sm.nan_from()[threadIdx.x] = nan_from;
    softmax_sync<S>();
    if (more) write_q<S, BF>(p, sm, q, (pc + 1) & 1);
    const int slot = (int)blockIdx.x + seg;  // workspace piece
    if (threadIdx.x < rows) {
      const int row = threadIdx.x, r = row % ROWS, g = row / ROWS;
      float sum[kStep], top = -INFINITY, all = 0.f;  // the row's denominator `all`, in units of 2^top
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        const int st = i * G + g;
        const float* x = sm.wred(st * 4) + r;
        sum[i] = (x[0] + x[ROWS]) + (x[2 * ROWS] + x[3 * ROWS]);
        if (sum[i] != 0.f) top = fmaxf(top, sm.base(st)[r]);
      }
      float wgt[kStep];
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        wgt[i] = sum[i] == 0.f ? 0.f : ex2(sm.base(i * G + g)[r] - top);
        if (wgt[i] != 0.f) all += sum[i] * wgt[i];
      }
      const float f = all > 0.f ? p.s.out_scale / all : all;  // 0 for a row without tokens, NaN for a NaN row
#pragma unroll
      for (int i = 0; i < kStep; ++i) sm.delta(i * G + g)[r] = wgt[i] == 0.f ? 0.f : wgt[i] * f;
      const float lse = all == 0.f ? -INFINITY : (top + __log2f(all)) * kLn2f;
      const size_t out_row = (size_t)(w.b * p.s.q_len + (row >> 2)) * p.s.hq + w.h * kGroup + (row & 3);
      if (!whole) p.s.ws_lse[(size_t)slot * p.s.rows_pad + row] = lse;
      else if (p.s.out_lse) p.s.out_lse[out_row] = lse;
    }
#pragma unroll
    for (int x = 0; x < S::LANES; ++x) {  // each lane's last product (it may have none in this piece)
      const int last = ((blk + nblk) * S::UNITS - 1 - x) / S::LANES * S::LANES + x;
      if (last >= blk * S::UNITS && last < (blk + nblk) * S::UNITS)
        mbar_wait_bounded(sm.bar(Smem<S>::P_DONE, sm.pi(x, last / S::LANES)), (uint32_t)(last / S::LANES >> 1) & 1u, abort,
                          p.s.status);
    }
    tc_fence_after();
    softmax_sync<S>();
    if (tid < ROWS) base[tid] = 0.f;  // for the next piece
#pragma unroll
    for (int st = 0; st < W; ++st) nan_from = min(nan_from, sm.nan_from()[st * 128 + tid]);
    // this warpgroup's share of the rows: G * ROWS / 4 from row `stream` * that on
    constexpr int kShare = G * ROWS / W, kChunk = kShare < 4 ? kShare : 4;
#pragma unroll 1
    for (int c = stream * kShare; c < (stream + 1) * kShare; c += kChunk) {
      if (c >= rows) break;
      const int g = c / ROWS, r0 = c % ROWS;
      float o[kChunk];
#pragma unroll
      for (int r = 0; r < kChunk; ++r) o[r] = 0.f;
      uint32_t raw[kStep][kPParts][kChunk];
#pragma unroll
      for (int i = 0; i < kStep; ++i)
#pragma unroll
        for (int j = 0; j < kPParts; ++j) tmem_ld(lanes + (i * G + g) * S::PROW + j * ROWS + r0, raw[i][j]);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
#pragma unroll
        for (int r = 0; r < kChunk; ++r) {
          float x = __uint_as_float(raw[i][kPParts - 1][r]);
#pragma unroll
          for (int j = kPParts - 2; j >= 0; --j)
            x = fmaf(x, j == kPParts - 2 ? 1.f / kLastPart : 1.f / 32.f, __uint_as_float(raw[i][j][r]));
          const float f = sm.delta(i * G + g)[r0 + r];
          if (f != 0.f) o[r] = fmaf(x, f, o[r]);  // a stream without tokens may hold anything
        }
      }
#pragma unroll
      for (int r = 0; r < kChunk; ++r) {
        const int row = c + r;
        // draft row / 4 sees the tokens before min(len, first + row / 4)
        if (nan_from < piece.first + (row >> 2)) o[r] = __int_as_float(0x7fffffff);
        if (row < rows) {
          const size_t out_row = (size_t)(w.b * p.s.q_len + (row >> 2)) * p.s.hq + w.h * kGroup + (row & 3);
          if (!whole) p.s.ws_o[((size_t)slot * p.s.rows_pad + row) * kHeadDim + tid] = o[r];
          else if (p.s.out_o) p.s.out_o[out_row * kHeadDim + tid] = o[r];
          else reinterpret_cast<uint16_t*>(p.s.out)[out_row * kHeadDim + tid] = (uint16_t)(pack2<BF>(o[r], 0.f) & 0xffffu);
        }
      }
    }
    tc_fence_before();  // O is read before the next piece's first product overwrites it
    softmax_sync<S>();     // and so is all that the streams share
    blk += nblk;
    ++pc;
  });
}

template <class S, bool MASK>
__device__ __forceinline__ float unit_weight(uint32_t slot, const float* base, float kc, int late, int row0) {
  float sum = 0.f;
#pragma unroll
  for (int c = 0; c < S::ROWS; c += 8) {
    float s[8];
    read_scores<S>(slot, c, s);
#pragma unroll
    for (int r = 0; r < 8; r += 4) {
      const float4 b4 = *reinterpret_cast<const float4*>(base + c + r);
      const float bb[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = fmaf(s[r + i], kc, bb[i]);
        if (MASK && late >= (row0 + c + r + i) >> 2) x = -INFINITY;
        sum += ex2(x);
      }
    }
  }
  return sum;
}

// A warpgroup takes every fourth block, all its row groups.
template <class S, bool BF>
__device__ void weigh(const ScaledTcParams& p, const Schedule& sch, const Smem<S>& sm, uint32_t tmem, volatile int* abort) {
  constexpr int G = S::G;
  const int stream = threadIdx.x >> 7;
  const int tid = threadIdx.x & 127, warp = tid >> 5, lane = tid & 31;
  const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
  const int rows = kGroup * p.s.q_len;
  auto row_lse = [&](int b, int h) {  // -lse in base 2; -inf (weight 0) for padding and rows without tokens
    const int row = threadIdx.x;
    if (row >= rows) return -INFINITY;
    const float v = __ldcg(p.lse + (size_t)(b * p.s.q_len + (row >> 2)) * p.s.hq + h * kGroup + (row & 3));
    return v == -INFINITY ? -INFINITY : -v * 1.4426950408889634f;
  };
  int blk = 0, pc = 0;
  for_pieces(p.s, sch, [&](const SegWalk& w, int, int n) {
    const int seg_end = w.seg_start + w.pages;
    const Piece piece = piece_of(p.s, w);
    if (pc == 0) {
      QItem<S> q;
      load_q<S, BF>(p, sm, w.b, w.h, q);
      if (threadIdx.x < G * S::ROWS) sm.base(0)[threadIdx.x] = row_lse(w.b, w.h);
      softmax_sync<S>();
      write_q<S, BF>(p, sm, q, 0);
      softmax_sync<S>();
    }
    const float cq = sm.cq()[pc & 1];
    const int nblk = blocks_of(n);
    for (int k = (stream - blk) & (S::W - 1); k < nblk; k += S::W) {
      const int bk = blk + k;
      const int np = min(kBlockPages, n - k * kBlockPages);
      const int tok0 = (w.pg + k * kBlockPages) * kPageSize;
      const int tok = tok0 + tid;
      const float4 meta = read_meta(p, sm, bk, abort);
      const float kc = meta.x * cq;
      const int id = __float_as_int(meta.w);
      const bool held = tid < np * kPageSize && tok < piece.len;
      float* const at = p.scores + ((size_t)max(id, 0) * p.s.hkv + w.h) * kPageSize + (tid & 15);
      const float old = (held && id >= 0 && tok < piece.fresh) ? __ldcg(at) : 0.f;  // in flight during the score product
      const bool masked = np < kBlockPages || tok0 + kBlock > piece.first || tok0 + kBlock > piece.len;
      // draft qi sees the token iff late < qi.  Of a token that no draft sees the padding rows must not see it
      // either: their scores are 0 times its K, NaN for a K or a scale that is not finite.
      const int late = held && tok - piece.first < p.s.q_len - 1 ? tok - piece.first : 0x7fffffff;
      float sum = 0.f;
#pragma unroll 1
      for (int g = 0; g < G; ++g) {
        const int u = bk * G + g;
        mbar_wait_bounded(sm.bar(Smem<S>::S_FULL, u % S::NS), (uint32_t)(u / S::NS) & 1u, abort, p.s.status);
        tc_fence_after();
        const uint32_t slot = lanes + (u % S::NS) * S::STRIDE;
        sum += masked ? unit_weight<S, true>(slot, sm.base(0) + g * S::ROWS, kc, late, g * S::ROWS)
                      : unit_weight<S, false>(slot, sm.base(0) + g * S::ROWS, kc, late, g * S::ROWS);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sm.bar(Smem<S>::S_EMPTY, u % S::NS));
      }
      if (held && id >= 0) *at = old + sum;
    }
    if (seg_end < sch.end) {  // the next piece's Q and rows
      SegWalk nw = w;
      next_segment(p.s, nw);
      QItem<S> q;
      load_q<S, BF>(p, sm, nw.b, nw.h, q);
      const float x = threadIdx.x < G * S::ROWS ? row_lse(nw.b, nw.h) : 0.f;
      softmax_sync<S>();
      write_q<S, BF>(p, sm, q, (pc + 1) & 1);
      if (threadIdx.x < G * S::ROWS) sm.base(0)[threadIdx.x] = x;
      softmax_sync<S>();
    }
    blk += nblk;
    ++pc;
  });
}

template <class S, bool BF>
__global__ void __launch_bounds__(S::THREADS, 1)
    sqa_scaled_tc_kernel(const ScaledTcParams p, const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v) {
  extern __shared__ uint8_t smem_raw[];
  // an offset, not a cast of an aligned address: the compiler keeps seeing shared memory
  const Smem<S> sm{smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u)};
  const int tiles = p.s.num_stages;
  const int warp = threadIdx.x >> 5;
  constexpr int kScoreWarp = S::SOFTMAX / 32, kValueWarp = kScoreWarp + 1, kProducerWarp = kScoreWarp + 2,
                kMetaWarp = kScoreWarp + 3;
  if (threadIdx.x == 0) {
    for (int i = 0; i < tiles; ++i) {
      mbar_init(sm.bar(Smem<S>::FULL, i), 1);
      mbar_init(sm.bar(Smem<S>::EMPTY, i), 1);
    }
    for (int i = 0; i < 8; ++i) {
      mbar_init(sm.bar(Smem<S>::S_FULL, i), 1);
      mbar_init(sm.bar(Smem<S>::S_EMPTY, i), 4 * S::GP);
    }
    for (int i = 0; i < 2 * S::LANES; ++i) {
      mbar_init(sm.bar(Smem<S>::P_FULL, i), 4 * S::GP);
      mbar_init(sm.bar(Smem<S>::P_DONE, i), 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(sm.bar(Smem<S>::Q_READY, i), S::SOFTMAX / 32);
    for (int i = 0; i < kMetaSlots; ++i) {
      mbar_init(sm.bar(Smem<S>::M_FULL, i), 1);
      mbar_init(sm.bar(Smem<S>::M_EMPTY, i), S::ATTEND ? 4 * S::G : 4);  // the warps that read a block's scales
    }
    mbar_init(sm.bar(Smem<S>::DONE), S::ATTEND ? 2 : 1);  // one commit from each issuer
    fence_mbar_init();
  }
  if (warp == kProducerWarp && (threadIdx.x & 31) == 0) {
    prefetch_tensormap(&tm_k);
    if (S::ATTEND) prefetch_tensormap(&tm_v);
  }
  // The value issuer has nothing to do before the first P: it prefetches the CTA's first
  // pages into L2 before the dependency wait (hints only).
  if (warp == kValueWarp) prefetch_start<S::F8, S::ATTEND>(p.s, &tm_k, &tm_v, tiles / S::TILES * kBlockPages);
  grid_dependency_wait();
  allow_dependent_launch();
  if (warp == kScoreWarp) {
    tmem_alloc(smem_u32(sm.tmem()), 512);
    tmem_relinquish();
  }
  if (warp == 0) build_schedule(p.s, sm.sch());
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *sm.tmem();
  const Schedule sch = *sm.sch();
  volatile int* abort = &sm.sch()->abort;
  if (warp == kProducerWarp) {
    produce<S>(p, sch, &tm_k, &tm_v, sm, tiles, abort);
  } else if (warp == kMetaWarp) {
    page_meta<S>(p, sch, sm, abort);
  } else if (warp == kScoreWarp) {
    issue_scores<S, BF>(p, sch, sm, tmem, tiles, abort);
  } else if (warp == kValueWarp) {
    if constexpr (S::ATTEND) issue_values<S>(p, sch, sm, tmem, tiles, abort);
  } else {
    if constexpr (S::ATTEND) attend<S, BF>(p, sch, sm, tmem, tiles, abort);
    else weigh<S, BF>(p, sch, sm, tmem, abort);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kScoreWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------ merge of split segments
// As sqa_segment_merge_kernel (one warp a row, 4 rows a CTA), with a NaN part making the row NaN.
__global__ void __launch_bounds__(128) sqa_scaled_merge_kernel(const MergeParams p) {
  allow_dependent_launch();
  const int s = blockIdx.x;
  const int b = s / p.hkv, h = s - b * p.hkv;
  const int2 info = p.seg_split
                        ? aligned_segment_pieces(p.seq_lens, p.max_pages, p.hkv, p.seg_split, b, h)
                        : segment_pieces(p.seq_lens, p.batch, p.max_pages, p.hkv, p.seg_cost, p.split_grid, b, h);
  grid_dependency_wait();
  const int row = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (row >= kGroup * p.q_len || info.y == 1) return;  // one piece: written by the split kernel
  const int lane = threadIdx.x & 31;
  const size_t out_row = (size_t)(b * p.q_len + (row >> 2)) * p.hq + h * kGroup + (row & 3);
  __half* out = p.out ? p.out + out_row * kHeadDim : nullptr;
  float* out_o = p.out_o ? p.out_o + out_row * kHeadDim : nullptr;
  float* out_lse = p.out_lse ? p.out_lse + out_row : nullptr;
  const size_t first = (size_t)info.x * p.piece_rows + row;
  bool nan = false;
  for (int i = lane; i < info.y; i += 32) {
    const float l = __ldg(p.parts_lse + first + (size_t)i * p.piece_rows);
    nan |= l != l;
  }
  if (info.y == 0) {  // no page: nothing is visible
    if (out) reinterpret_cast<uint2*>(out)[lane] = make_uint2(0u, 0u);
    if (out_o) reinterpret_cast<float4*>(out_o)[lane] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (out_lse && lane == 0) *out_lse = -INFINITY;
    return;
  }
  merge_row<false>(p.parts_o + first * kHeadDim, (size_t)p.piece_rows * kHeadDim, p.parts_lse + first,
                   (size_t)p.piece_rows, info.y, out, out_o, out_lse, p.bf16 != 0);
  if (__any_sync(0xffffffffu, nan)) {
    const float x = __int_as_float(0x7fffffff);
    if (out) reinterpret_cast<uint2*>(out)[lane] = make_uint2(0x7fff7fffu, 0x7fff7fffu);  // NaN in fp16 and bf16
    if (out_o) reinterpret_cast<float4*>(out_o)[lane] = make_float4(x, x, x, x);
    if (out_lse && lane == 0) *out_lse = x;
  }
}

// ------------------------------------------------------------------ launch
constexpr int kMaxSmem = 227 * 1024;

template <class S>
constexpr int tiles_that_fit() {
  constexpr int n = (kMaxSmem - 1024 - Smem<S>::RING) / kTileBytes;
  constexpr int tiles = (n < Smem<S>::kMaxTiles ? n : Smem<S>::kMaxTiles) / S::TILES * S::TILES;
  static_assert(tiles / 2 > S::W / S::G, "the ring holds more blocks than a stream skips");
  return tiles;
}

template <class S, bool BF>
cudaError_t launch_shape(ScaledTcParams& p, const CUtensorMap& tm_k, const CUtensorMap& tm_v, int grid,
                         cudaStream_t stream) {
  auto kernel = sqa_scaled_tc_kernel<S, BF>;
  p.s.num_stages = tiles_that_fit<S>();
  const int smem = 1024 + Smem<S>::RING + p.s.num_stages * kTileBytes;
  static std::atomic<bool> configured[64];  // per device
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err != cudaSuccess) return err;
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(S::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  err = cudaLaunchKernelEx(&cfg, kernel, p, tm_k, tm_v);
  return err != cudaSuccess ? err : cudaGetLastError();
}

template <int PARTS, bool ATTEND, bool BF>
cudaError_t launch_rows(ScaledTcParams& p, const CUtensorMap& tm_k, const CUtensorMap& tm_v, int grid,
                        cudaStream_t stream) {
  const int rows = kGroup * p.s.q_len;
  if constexpr (ATTEND) {
    if (rows <= 8) return launch_shape<Shape<PARTS, 8, 1, 2, true>, BF>(p, tm_k, tm_v, grid, stream);
    if (rows <= 16) return launch_shape<Shape<PARTS, 16, 1, 2, true>, BF>(p, tm_k, tm_v, grid, stream);
    if (rows <= 32) return launch_shape<Shape<PARTS, 16, 2, 2, true>, BF>(p, tm_k, tm_v, grid, stream);
    return launch_shape<Shape<PARTS, 16, 4, 4, true>, BF>(p, tm_k, tm_v, grid, stream);
  } else {  // wider units: no P, no O, and K read less often
    if (rows <= 8) return launch_shape<Shape<PARTS, 8, 1, 4, false>, BF>(p, tm_k, tm_v, grid, stream);
    if (rows <= 16) return launch_shape<Shape<PARTS, 16, 1, 4, false>, BF>(p, tm_k, tm_v, grid, stream);
    if (rows <= 32) return launch_shape<Shape<PARTS, 32, 1, 4, false>, BF>(p, tm_k, tm_v, grid, stream);
    // three parts of 32 rows leave four slots: two for each of two warpgroups
    return launch_shape<Shape<PARTS, 32, 2, PARTS == 3 ? 2 : 4, false>, BF>(p, tm_k, tm_v, grid, stream);
  }
}

ScaledTcParams tc_params(const ScaledParams& p) {
  ScaledTcParams t = {};
  t.s.q = static_cast<const __half*>(p.q);
  t.s.block_tables = p.block_tables;
  t.s.seq_lens = p.seq_lens;
  t.s.mask_lens = p.mask_lens;
  t.s.shard_lens = p.mask_lens != nullptr;
  t.s.out = static_cast<__half*>(p.out);
  t.s.out_o = p.out_o;
  t.s.out_lse = p.out_lse;
  t.s.ws_o = p.ws_o;
  t.s.ws_lse = p.ws_lse;
  t.s.status = p.status;
  t.s.batch = p.batch;
  t.s.q_len = p.q_len;
  t.s.hq = p.hq;
  t.s.hkv = p.hkv;
  t.s.max_pages = p.max_pages;
  t.s.num_pages = p.num_pages;
  t.s.rows_pad = p.rows_pad;
  t.s.scale_log2 = p.scale_log2;
  t.s.bf16 = p.bf16;
  t.s.hnd = p.hnd;
  t.s.out_scale = p.out_scale;
  t.s.seg_cost = p.seg_cost;
  t.s.seg_split = p.seg_split;
  t.k_scales = p.k_scales;
  t.v_scales = p.v_scales;
  t.scale_stride = p.scale_stride;
  t.lse = p.lse;
  t.scores = p.scores;
  return t;
}

}  // namespace

cudaError_t launch_scaled_attention(const ScaledParams& p, const CUtensorMap& tm_k, const CUtensorMap& tm_v,
                                    cudaStream_t stream) {
  ScaledTcParams t = tc_params(p);
  cudaError_t err = p.bf16 ? launch_rows<2, true, true>(t, tm_k, tm_v, p.grid, stream)
                           : launch_rows<3, true, false>(t, tm_k, tm_v, p.grid, stream);
  if (err != cudaSuccess || p.seg_split == 1) return err;  // one CTA a segment: nothing to merge
  MergeParams m = {};
  m.parts_o = p.ws_o;
  m.parts_lse = p.ws_lse;
  m.seq_lens = p.seq_lens;
  m.out = static_cast<__half*>(p.out);
  m.out_o = p.out_o;
  m.out_lse = p.out_lse;
  m.piece_rows = p.rows_pad;
  m.batch = p.batch;
  m.q_len = p.q_len;
  m.hq = p.hq;
  m.hkv = p.hkv;
  m.max_pages = p.max_pages;
  m.bf16 = p.bf16;
  m.split_grid = p.grid;
  m.seg_cost = p.seg_cost;
  m.seg_split = p.seg_split;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.batch * p.hkv), (unsigned)p.q_len);  // 4 rows a CTA
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  err = cudaLaunchKernelEx(&cfg, sqa_scaled_merge_kernel, m);
  return err != cudaSuccess ? err : cudaGetLastError();
}

cudaError_t launch_weights(const ScaledParams& p, const CUtensorMap& tm_k, cudaStream_t stream) {
  ScaledTcParams t = tc_params(p);
  t.s.out = reinterpret_cast<__half*>(p.scores);  // only asked for being there: a length under q_len is reported
  if (p.k_scales != nullptr)
    return p.bf16 ? launch_rows<2, false, true>(t, tm_k, tm_k, p.grid, stream)
                  : launch_rows<3, false, false>(t, tm_k, tm_k, p.grid, stream);
  return p.bf16 ? launch_rows<0, false, true>(t, tm_k, tm_k, p.grid, stream)
                : launch_rows<0, false, false>(t, tm_k, tm_k, p.grid, stream);
}

}  // namespace sqa
