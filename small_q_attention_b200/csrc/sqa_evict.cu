// sqa_evict.cu -- eviction from the paged cache by accumulated attention weight.
//
// Per (sequence b, KV head h) with n = seq_lens[b] > budget, the kept tokens are the
// first `sinks`, the last `recent` and, of the others, the budget - sinks - recent
// with the highest score (NaN counts as the lowest; equal scores: the earlier token).
// They move, in order of position, to positions 0 .. budget - 1 of the same pages:
// K, V and score.  Every page of a block-scaled cache that is written gets the scale
// of the values that it now holds.  Sequences of at most `budget` tokens are left.
//
// A thread-block cluster of C CTAs works on one (b, h):
//
// 1. Selection.  Each CTA holds a slice of the scores as order-preserving 32-bit keys.
//    A radix search over the range [lo, hi] that still holds the wanted rank: 256 equal
//    bins, histograms exchanged over the cluster, one cluster barrier a pass.  The range is
//    taken from the scores themselves, so that the bins are used evenly (scores share their
//    leading bits; a fixed digit would send them all to one bin and serialise its counter).
//    Once the bin of the wanted rank holds at most 256 keys, every CTA gets them all
//    and each thread ranks one of them against the others: two exchanges for 8192 tokens
//    where bins alone took four (2900 cycles each).  More than 256 equal keys end in a
//    range of one key.
// 2. Ranks.  A kept token's target is a sum of counts of earlier slices (shared through
//    the cluster) and of a block scan; kept[] lists the kept positions.
// 3. Moves, in place and in waves of C x T / 32 target pages: a warp loads the 16 source rows
//    of its target page (K, V, scores, source scales) into registers, the cluster meets
//    at a barrier, then every warp writes its page.  A source is never before its
//    target, and the sources of later waves lie in pages behind this wave's targets, so
//    nothing is overwritten before it is read, and a wave's loads may be issued before the
//    last one's stores (done for e4m3, whose pages take half the registers).
//
// C and T are chosen so that every cluster is resident at once where that is possible: one CTA of
// 512 threads per SM, or two of 256.  (Clusters of 8 x 256 throughout: 4 x 8192 to 2048 33.5 us instead
// of 26.9, 32 x 7001 to 1500 in e4m3 151 instead of 63.)  An instrumented CTA selects for 12 us and
// moves for 8 in the first, 23 and 39 us in the second (floors of the whole: 10.7 and 27.9 us).
#include <mutex>

#include "small_q_attention.h"
#include "sqa_internal.h"
#include "sqa_ptx.cuh"
#include "sqa_scaled.cuh"

namespace sqa {
namespace {

constexpr int kBins = 256;
constexpr int kCandidates = 256;  // keys that are ranked directly
constexpr int kEvictMaxCluster = 8;
constexpr int kKeyCap = 12288;  // keys of a slice held in shared memory (48 KB); further ones are read again

struct EvictParams {
  uint8_t* k_cache;
  uint8_t* v_cache;
  float* k_scales;
  float* v_scales;
  float* scores;  // [num_pages, hkv, 16]
  const int32_t* block_tables;
  const int32_t* seq_lens;
  int32_t* new_lens;
  int32_t* kept;  // [batch, hkv, budget]
  unsigned int* status;
  long long page_stride;   // bytes
  long long scale_stride;  // floats
  int hkv, num_pages, max_pages, hnd;
  int budget, recent, sinks;
  int cluster, key_cap;
};

// What the CTAs of a cluster tell one another they store into each other's shared memory before
// a cluster barrier and read from their own after it: remote stores are not waited for, while a
// loop of remote loads cost 8 round trips (a radix pass took 4500 cycles with them).
template <int T>
struct EvictShared {
  unsigned int hist[kBins];                        // this slice's
  unsigned int hists[2][kEvictMaxCluster][kBins];  // every slice's, by pass parity
  unsigned int range[kEvictMaxCluster][2];         // every slice's (lowest, highest) key
  unsigned int counts[kEvictMaxCluster][2];        // every slice's (above, equal)
  unsigned int cand_key[kCandidates], cand_pos[kCandidates];
  unsigned int warp_a[T / 32], warp_b[T / 32];
  unsigned int pick[4];
  unsigned int fill;
};

// `v` to the same shared-memory location of the CTA of rank `rank`.
__device__ __forceinline__ void st_cluster_u32(void* p, int rank, unsigned int v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_map(smem_u32(p), (uint32_t)rank)), "r"(v) : "memory");
}

// Order-preserving key of a score; NaN lowest, the two zeros equal.
__device__ __forceinline__ unsigned int score_key(float f) {
  if (f != f) return 0u;
  const unsigned int u = __float_as_uint(f == 0.f ? 0.f : f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// The page that the warp holds (load i, row i * kRows + sub, 16 elements a lane; row r's scale in lane r) at
// the scale of what it now holds, which is returned.  Whole warp.  Maxima are taken in fp16, which
// holds every e4m3 number; with power-of-two scales, as the append and this kernel leave them, so
// is the product (a factor of 2^-14..2^14; what falls below fp16's range is zero in e4m3 as
// well), and rows that keep their scale are not touched.  Any other scale goes through fp32.
template <int kLoads, int kRows>
__device__ __forceinline__ float rescale_page(uint4 (&x)[kLoads], float source, int sub) {
  float amax = 0.f, s[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    s[i] = __shfl_sync(0xffffffffu, source, i * kRows + sub);
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    __half2 m = __floats2half2_rn(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      m = __hmax2(m, __hmax2(__habs2(half2_of_e4m3x2(w[c] & 0xffffu)), __habs2(half2_of_e4m3x2(w[c] >> 16))));
    const float2 f = __half22float2(m);
    amax = fmaxf(amax, finite_abs(fmaxf(f.x, f.y) * s[i]));
  }
  const float scale = page_scale(warp_max(amax));
  const int e = (int)(__float_as_uint(scale) >> 23);
  bool plain = true;  // every row's factor is a power of two within fp16
  int shift[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const uint32_t u = __float_as_uint(s[i]);
    shift[i] = (int)(u >> 23) - e;
    plain = plain && (u & 0x7fffffu) == 0u && abs(shift[i]) <= 14;
    if (s[i] == 0.f) {  // rows of zeros, or none
      shift[i] = 0;
      plain = plain && (x[i].x | x[i].y | x[i].z | x[i].w) == 0u;
    }
  }
  if (__all_sync(0xffffffffu, plain)) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      if (shift[i] == 0) continue;
      const __half2 f = __float2half2_rn(__uint_as_float((uint32_t)(shift[i] + 127) << 23));
      uint32_t* const w = reinterpret_cast<uint32_t*>(&x[i]);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        w[c] = e4m3x2_of_half2(__hmul2(half2_of_e4m3x2(w[c] & 0xffffu), f)) |
               (e4m3x2_of_half2(__hmul2(half2_of_e4m3x2(w[c] >> 16), f)) << 16);
    }
  } else {
    const float inv = 1.f / scale;  // a power of two: multiplying by it is dividing by scale
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      uint32_t* const w = reinterpret_cast<uint32_t*>(&x[i]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float2 a = unpack_e4m3x2(w[c]), d = unpack_e4m3x2(w[c] >> 16);
        w[c] = pack_e4m3x4(a.x * s[i] * inv, a.y * s[i] * inv, d.x * s[i] * inv, d.y * s[i] * inv);
      }
    }
  }
  return scale;
}

// E: bytes per cached element, 2 (16-bit) or 1 (block-scaled e4m3); T threads.
template <int E, int T>
__global__ void __launch_bounds__(T, 512 / T) sqa_cache_evict_kernel(const EvictParams p) {
  constexpr int kWarps = T / 32;
  extern __shared__ unsigned int keys[];  // key_cap
  __shared__ EvictShared<T> sh;
  grid_dependency_wait();
  allow_dependent_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = p.cluster;
  const int rank = (int)blockIdx.x % C;
  const int seg = (int)blockIdx.x / C;
  const int b = seg / p.hkv, h = seg - b * p.hkv;
  const int len = __ldg(p.seq_lens + b);
  const int32_t* table = p.block_tables + (size_t)b * p.max_pages;
  auto meet = [&]() {  // barrier of the cluster
    if (C > 1) cluster_sync_all();
    else __syncthreads();
  };
  int32_t* const kept = p.kept + (size_t)seg * p.budget;

  // Sequences that stay as they are: short ones, and those whose length or pages are bad.
  unsigned int err = 0;
  const int pages = page_count(len);
  if (len < 0) err = 4u;                 // SQA_DEV_SEQ_TOO_SHORT
  else if (pages > p.max_pages) err = 2u;  // SQA_DEV_SEQ_TOO_LONG
  else if (len > p.budget) {
    int bad = 0;
    for (int i = tid; i < pages; i += T) {
      const int id = __ldg(table + i);
      bad |= id < 0 || id >= p.num_pages;
    }
    if (__syncthreads_or(bad)) err = 8u;  // SQA_DEV_BAD_PAGE
  }
  if (err || len <= p.budget) {  // the same for every CTA of the cluster
    for (int i = rank * T + tid; i < p.budget; i += C * T)
      kept[i] = (!err && i < len) ? i : -1;
    if (h == 0 && rank == 0 && tid == 0) {
      p.new_lens[b] = len;
      if (err && p.status) atomicOr(p.status, err);
    }
    return;
  }
  if (h == 0 && rank == 0 && tid == 0) p.new_lens[b] = p.budget;

  __syncwarp();
  if (C > 1) cluster_arrive_all();  // this CTA runs: the others may store into its shared memory
  // ---- 1. the key of the last score that is kept
  const int middle = len - p.sinks - p.recent;  // candidates
  const int want = p.budget - p.sinks - p.recent;
  const int per = (middle + C - 1) / C;
  const int a0 = p.sinks + min(middle, rank * per);
  const int count = p.sinks + min(middle, (rank + 1) * per) - a0;
  const int off = a0 & 3;  // keys[] starts at a multiple of four positions: 16-byte loads of the scores
  auto scores_of = [&](int t) { return p.scores + ((size_t)__ldg(table + t / kPageSize) * p.hkv + h) * kPageSize + t % kPageSize; };
  // f(i, key) for i = from, from + step, .. < to.  One loop over shared memory where it holds the whole
  // slice: with the choice inside, no two iterations overlapped.
  const bool held = off + count <= p.key_cap;
  auto for_keys = [&](int from, int to, int step, auto f) {
    if (held) {
#pragma unroll 4
      for (int i = from; i < to; i += step) f(i, keys[i + off]);
    } else {
#pragma unroll 1
      for (int i = from; i < to; i += step)
        f(i, i + off < p.key_cap ? keys[i + off] : score_key(__ldcg(scores_of(a0 + i))));
    }
  };
  unsigned int lo = 0xffffffffu, hi = 0u;
  constexpr int kAhead = 4;  // loads in flight: page ids, then scores
  for (int q0 = tid; q0 < (off + count + 3) / 4; q0 += kAhead * T) {
    float4 f[kAhead];
    const float* src[kAhead];
#pragma unroll
    for (int c = 0; c < kAhead; ++c) {
      const int q = q0 + c * T;
      src[c] = q < (off + count + 3) / 4 ? scores_of(a0 - off + 4 * q) : nullptr;
    }
#pragma unroll
    for (int c = 0; c < kAhead; ++c)
      f[c] = src[c] ? __ldcg(reinterpret_cast<const float4*>(src[c])) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kAhead; ++c) {
      if (!src[c]) continue;
      const unsigned int k[4] = {score_key(f[c].x), score_key(f[c].y), score_key(f[c].z), score_key(f[c].w)};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = 4 * (q0 + c * T) + i;
        if (at < p.key_cap) keys[at] = k[i];
        if (at >= off && at < off + count) {
          lo = min(lo, k[i]);
          hi = max(hi, k[i]);
        }
      }
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) {
    sh.warp_a[warp] = lo;
    sh.warp_b[warp] = hi;
  }
  __syncthreads();
  if (C > 1) cluster_wait_all();  // every CTA of the cluster runs
  if (tid < C) {  // this slice's range to CTA `tid`
    lo = sh.warp_a[0];
    hi = sh.warp_b[0];
    for (int w = 1; w < kWarps; ++w) {
      lo = min(lo, sh.warp_a[w]);
      hi = max(hi, sh.warp_b[w]);
    }
    st_cluster_u32(&sh.range[rank][0], tid, lo);
    st_cluster_u32(&sh.range[rank][1], tid, hi);
  }
  meet();
  lo = 0xffffffffu;
  hi = 0u;
  for (int r = 0; r < C; ++r) {
    lo = min(lo, sh.range[r][0]);
    hi = max(hi, sh.range[r][1]);
  }
  // Kept: every key > last, and of the keys == last the first `need`.
  // Invariant: want - need keys lie above hi, and at least `need` in [lo, hi].
  int need = want;
  bool ranked = want == 0;  // last and need are final
  unsigned int last = hi;
  for (int pass = 0; !ranked && lo < hi; ++pass) {
    const int shift = max(0, 24 - __clz(hi - lo));  // (hi - lo) >> shift < 256
    if (tid < kBins) sh.hist[tid] = 0u;
    if (tid == 0) sh.fill = 0u;
    __syncthreads();
    for_keys(tid, count, T, [&](int, unsigned int k) {
      if (k >= lo && k <= hi) atomicAdd(&sh.hist[(k - lo) >> shift], 1u);
    });
    __syncthreads();
    if (tid < kBins) {
      const unsigned int mine = sh.hist[tid];
#pragma unroll
      for (int r = 0; r < kEvictMaxCluster; ++r)
        if (r < C) st_cluster_u32(&sh.hists[pass & 1][rank][tid], r, mine);
    }
    meet();  // also: every CTA has read the pass before the last
    // thread t < 256: bin 255 - t, so that an inclusive scan counts from the top
    const int bin = kBins - 1 - tid;
    unsigned int n = 0, incl = 0;
    if (tid < kBins) {
#pragma unroll
      for (int r = 0; r < kEvictMaxCluster; ++r)
        if (r < C) n += sh.hists[pass & 1][r][bin];
      incl = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const unsigned int y = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += y;
      }
      if (lane == 31) sh.warp_a[warp] = incl;
    }
    __syncthreads();
    if (tid < kBins) {
      for (int w = 0; w < warp; ++w) incl += sh.warp_a[w];
      if (incl >= (unsigned int)need && incl - n < (unsigned int)need) {  // exactly one thread
        sh.pick[0] = (unsigned int)bin;
        sh.pick[1] = incl - n;  // keys above the bin, in the range
        sh.pick[2] = n;
      }
    }
    __syncthreads();
    const unsigned int j = sh.pick[0], total = sh.pick[2];
    const unsigned int edge = lo + (j << shift);
    hi = edge + min(hi - edge, (1u << shift) - 1u);
    lo = edge;
    need -= (int)sh.pick[1];
    if (lo < hi && total <= kCandidates) {
      // the bin's keys, with their positions, to every CTA, slice by slice
      unsigned int at = 0;
      for (int r = 0; r < rank; ++r) at += sh.hists[pass & 1][r][j];
      for_keys(tid, count, T, [&](int i, unsigned int k) {
        if (k >= lo && k <= hi) {
          const unsigned int c = at + atomicAdd(&sh.fill, 1u);
          for (int r = 0; r < C; ++r) {
            st_cluster_u32(&sh.cand_key[c], r, k);
            st_cluster_u32(&sh.cand_pos[c], r, (unsigned int)(a0 + i));
          }
        }
      });
      meet();
      if (tid < (int)total) {  // its rank: keys above it, and equal ones before it
        const unsigned int k = sh.cand_key[tid], t = sh.cand_pos[tid];
        int more = 0, before = 0;
#pragma unroll 4
        for (int c = 0; c < (int)total; ++c) {
          const unsigned int kc = sh.cand_key[c];
          more += kc > k;
          before += kc == k && sh.cand_pos[c] < t;
        }
        if (more + before == need - 1) {  // the last that is kept: exactly one
          sh.pick[0] = k;
          sh.pick[3] = (unsigned int)(before + 1);
        }
      }
      __syncthreads();
      last = sh.pick[0];
      need = (int)sh.pick[3];
      ranked = true;
    }
  }
  if (want == 0) need = 0;
  else if (!ranked) last = lo;

  // ---- 2. ranks: each thread a run of tokens (of odd length: no bank is met twice), one scan
  const int run = ((count + T - 1) / T) | 1;
  const int i0 = min(count, tid * run), i1 = min(count, i0 + run);
  unsigned int gt = 0, eq = 0;
  for_keys(i0, i1, 1, [&](int, unsigned int k) {
    gt += k > last;
    eq += k == last;
  });
  unsigned int gt_to = gt, eq_to = eq;  // up to and with this thread's
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const unsigned int x = __shfl_up_sync(0xffffffffu, gt_to, off), y = __shfl_up_sync(0xffffffffu, eq_to, off);
    if (lane >= off) {
      gt_to += x;
      eq_to += y;
    }
  }
  __syncthreads();  // warp_a is free
  if (lane == 31) {
    sh.warp_a[warp] = gt_to;
    sh.warp_b[warp] = eq_to;
  }
  __syncthreads();
  unsigned int all_gt = 0, all_eq = 0;
  unsigned int g = gt_to - gt, e = eq_to - eq;  // kept and equal tokens before this thread's
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) {
      g += all_gt;
      e += all_eq;
    }
    all_gt += sh.warp_a[w];
    all_eq += sh.warp_b[w];
  }
  if (C > 1) {
    if (tid < C) {
      st_cluster_u32(&sh.counts[rank][0], tid, all_gt);
      st_cluster_u32(&sh.counts[rank][1], tid, all_eq);
    }
    meet();
    for (int r = 0; r < rank; ++r) {
      g += sh.counts[r][0];
      e += sh.counts[r][1];
    }
  }
  for_keys(i0, i1, 1, [&](int i, unsigned int k) {
    const bool is_gt = k > last, is_eq = k == last;
    if (is_gt || (is_eq && e < (unsigned int)need)) kept[p.sinks + g + min(e, (unsigned int)need)] = a0 + i;
    g += is_gt;
    e += is_eq;
  });
  for (int i = rank * T + tid; i < p.sinks; i += C * T) kept[i] = i;
  for (int i = rank * T + tid; i < p.recent; i += C * T)
    kept[p.budget - p.recent + i] = len - p.recent + i;
  meet();  // kept[] is complete, for every CTA of the cluster

  // ---- 3. moves, C x T / 32 target pages a wave
  constexpr int kLanesPerRow = kHeadDim * E / 16;     // 16 (16-bit) or 8 (e4m3) lanes hold a row
  constexpr int kRowsPerLoad = 32 / kLanesPerRow;     // rows a warp loads at once
  constexpr int kLoads = kPageSize / kRowsPerLoad;
  const int sub = lane / kLanesPerRow;
  const size_t head = p.hnd ? (size_t)h * kPageSize * kHeadDim * E : (size_t)h * kHeadDim * E;
  const size_t row = p.hnd ? (size_t)kHeadDim * E : (size_t)p.hkv * kHeadDim * E;  // bytes from slot to slot
  const size_t in_row = head + (lane % kLanesPerRow) * 16;
  const int targets = (p.budget + kPageSize - 1) / kPageSize;
  struct Page {  // a wave's page: where it goes, and what the lane holds of it
    int rows, to;
    uint4 k[kLoads], v[kLoads];
    float score, ks, vs;
  };
  auto indexes = [&](int base, Page& x, int& from, int& slot) {
    const int target = base + rank * kWarps + warp;
    x.rows = target < targets ? min(kPageSize, p.budget - target * kPageSize) : 0;
    x.to = from = slot = 0;
    if (x.rows > 0) {
      x.to = __ldg(table + target);
      if (lane < x.rows) {
        const int t = __ldcg(kept + target * kPageSize + lane);
        from = __ldg(table + t / kPageSize);
        slot = t % kPageSize;
      }
    }
  };
  auto load = [&](Page& x, int from, int slot) {
    x.score = x.ks = x.vs = 0.f;
    if (x.rows <= 0) return;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = i * kRowsPerLoad + sub;
      const int rf = __shfl_sync(0xffffffffu, from, r), rs = __shfl_sync(0xffffffffu, slot, r);
      const size_t at = (size_t)rf * p.page_stride + rs * row + in_row;
      x.k[i] = x.v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (r < x.rows) {
        x.k[i] = __ldcg(reinterpret_cast<const uint4*>(p.k_cache + at));
        x.v[i] = __ldcg(reinterpret_cast<const uint4*>(p.v_cache + at));
      }
    }
    if (lane < x.rows) {
      x.score = __ldcg(p.scores + ((size_t)from * p.hkv + h) * kPageSize + slot);
      if constexpr (E == 1) {
        x.ks = __ldcg(p.k_scales + (size_t)from * p.scale_stride + h);
        x.vs = __ldcg(p.v_scales + (size_t)from * p.scale_stride + h);
      }
    }
  };
  auto store = [&](Page& x) {
    if (x.rows <= 0) return;
    if constexpr (E == 1) {
      const float new_ks = rescale_page<kLoads, kRowsPerLoad>(x.k, x.ks, sub);
      const float new_vs = rescale_page<kLoads, kRowsPerLoad>(x.v, x.vs, sub);
      if (lane == 0) {
        p.k_scales[(size_t)x.to * p.scale_stride + h] = new_ks;
        p.v_scales[(size_t)x.to * p.scale_stride + h] = new_vs;
      }
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = i * kRowsPerLoad + sub;
      if (r < x.rows) {
        const size_t at = (size_t)x.to * p.page_stride + r * row + in_row;
        *reinterpret_cast<uint4*>(p.k_cache + at) = x.k[i];
        *reinterpret_cast<uint4*>(p.v_cache + at) = x.v[i];
      }
    }
    if (lane < x.rows) p.scores[((size_t)x.to * p.hkv + h) * kPageSize + lane] = x.score;
  };
  const int wave = C * kWarps;
  Page x;
  int from, slot;
  indexes(0, x, from, slot);
  load(x, from, slot);
  if (wave < targets) {
    Page ahead;  // its indexes (16-bit caches) or all of it (e4m3) while this wave's loads are under way
    indexes(wave, ahead, from, slot);
    for (int base = 0; base < targets; base += wave) {
      const bool more = base + wave < targets;
      if (E == 1 && more) load(ahead, from, slot);
      meet();  // every source of this wave has been read
      store(x);
      if (more) {
        if (E == 2) load(ahead, from, slot);
        x = ahead;
        if (base + 2 * wave < targets) indexes(base + 2 * wave, ahead, from, slot);
      }
    }
  } else {
    meet();
    store(x);
  }
}
// Clusters of C CTAs that can be resident at once (and, once per device, the kernel's shared-memory limit).
template <int E, int T>
int resident_clusters(int cluster) {
  static std::mutex mu;
  static int known[64][kEvictMaxCluster + 1] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::lock_guard<std::mutex> lock(mu);
  if (known[dev][cluster] != 0) return known[dev][cluster];
  auto kernel = sqa_cache_evict_kernel<E, T>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kKeyCap * (int)sizeof(unsigned int)) !=
      cudaSuccess) {
    (void)cudaGetLastError();
    return 0;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cluster);
  cfg.blockDim = dim3(T);
  cfg.dynamicSmemBytes = kKeyCap * sizeof(unsigned int);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    n = 0;
  }
  known[dev][cluster] = n;
  return n;
}

template <int E, int T>
cudaError_t launch_evict(EvictParams p, int segments, int cluster, cudaStream_t stream) {
  auto kernel = sqa_cache_evict_kernel<E, T>;
  p.cluster = cluster;
  const int64_t slice = ((int64_t)p.max_pages * kPageSize + cluster - 1) / cluster + 3;  // + its start's remainder
  p.key_cap = slice < kKeyCap ? (int)slice : kKeyCap;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(segments * cluster));
  cfg.blockDim = dim3(T);
  cfg.dynamicSmemBytes = p.key_cap * sizeof(unsigned int);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, p);
  return err != cudaSuccess ? err : cudaGetLastError();
}

// The largest clusters of 512-thread CTAs (one a SM) that are all resident at once; where even single
// CTAs are not, 256 threads (two a SM), in rounds if need be.
template <int E>
cudaError_t launch_evict_shape(const EvictParams& p, int segments, cudaStream_t stream) {
  for (int c = kEvictMaxCluster; c >= 1; c /= 2)
    if (resident_clusters<E, 512>(c) >= segments) return launch_evict<E, 512>(p, segments, c, stream);
  (void)resident_clusters<E, 256>(1);  // sets the shared-memory limit
  return launch_evict<E, 256>(p, segments, 1, stream);
}

bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + (uintptr_t)b_bytes && y < x + (uintptr_t)a_bytes;
}

}  // namespace
}  // namespace sqa

using namespace sqa;

extern "C" SQA_API int sqa_cache_evict(const sqa_evict_args* a, const sqa_scales* scales, void* stream) {
  if (a == nullptr) return SQA_ERR_INVALID_ARGUMENT;
  if (a->head_dim != kHeadDim || a->page_size != kPageSize) return SQA_ERR_UNSUPPORTED;
  if (a->batch < 0 || a->num_kv_heads <= 0 || a->num_pages <= 0 || a->max_pages <= 0) return SQA_ERR_INVALID_ARGUMENT;
  if (a->kv_layout != SQA_KV_NHD && a->kv_layout != SQA_KV_HND) return SQA_ERR_UNSUPPORTED;
  if (a->kv_dtype != SQA_KV_SAME && a->kv_dtype != SQA_KV_FP8_E4M3) return SQA_ERR_UNSUPPORTED;
  const bool fp8 = a->kv_dtype == SQA_KV_FP8_E4M3;
  if (fp8 != (scales != nullptr)) return SQA_ERR_INVALID_ARGUMENT;  // e4m3 caches carry their scales
  if (a->budget < 1 || a->recent < 0 || a->sinks < 0 || (int64_t)a->recent + a->sinks > a->budget)
    return SQA_ERR_INVALID_ARGUMENT;
  if (a->page_stride < 0 || (a->page_stride > 0 && (a->page_stride < (int64_t)kPageSize * a->num_kv_heads * kHeadDim ||
                                                    a->page_stride % (fp8 ? 16 : 8) != 0)))
    return SQA_ERR_INVALID_ARGUMENT;
  if (scales && (scales->page_stride < 0 || (scales->page_stride > 0 && scales->page_stride < a->num_kv_heads)))
    return SQA_ERR_INVALID_ARGUMENT;
  // positions and grid sizes are 32-bit
  if (a->max_pages > (1 << 26) || a->budget > (1 << 30) || (int64_t)a->batch * a->num_kv_heads > (1 << 27))
    return SQA_ERR_UNSUPPORTED;
  if (a->batch == 0) return SQA_OK;
  if (!a->key_cache || !a->value_cache || !a->scores || !a->block_tables || !a->seq_lens || !a->new_lens || !a->kept ||
      (scales && (!scales->key || !scales->value)))
    return SQA_ERR_INVALID_ARGUMENT;
  // CTAs read lengths and tables while others write their results
  const int64_t lens = 4 * (int64_t)a->batch, tables = lens * a->max_pages, kept = lens * a->num_kv_heads * a->budget;
  if (overlap(a->new_lens, lens, a->seq_lens, lens) || overlap(a->new_lens, lens, a->block_tables, tables) ||
      overlap(a->kept, kept, a->seq_lens, lens) || overlap(a->kept, kept, a->block_tables, tables) ||
      overlap(a->kept, kept, a->new_lens, lens))
    return SQA_ERR_INVALID_ARGUMENT;
  const uintptr_t wide = reinterpret_cast<uintptr_t>(a->key_cache) | reinterpret_cast<uintptr_t>(a->value_cache) |
                         reinterpret_cast<uintptr_t>(a->scores);
  uintptr_t narrow = reinterpret_cast<uintptr_t>(a->block_tables) |
                     reinterpret_cast<uintptr_t>(a->seq_lens) | reinterpret_cast<uintptr_t>(a->new_lens) |
                     reinterpret_cast<uintptr_t>(a->kept) | reinterpret_cast<uintptr_t>(a->status);
  if (scales) narrow |= reinterpret_cast<uintptr_t>(scales->key) | reinterpret_cast<uintptr_t>(scales->value);
  if ((wide & 15u) || (narrow & 3u)) return SQA_ERR_INVALID_ARGUMENT;

  EvictParams p = {};
  const int elem = fp8 ? 1 : 2;
  p.k_cache = static_cast<uint8_t*>(a->key_cache);
  p.v_cache = static_cast<uint8_t*>(a->value_cache);
  p.k_scales = scales ? scales->key : nullptr;
  p.v_scales = scales ? scales->value : nullptr;
  p.scores = a->scores;
  p.block_tables = a->block_tables;
  p.seq_lens = a->seq_lens;
  p.new_lens = a->new_lens;
  p.kept = a->kept;
  p.status = a->status;
  p.page_stride = (a->page_stride > 0 ? a->page_stride : (int64_t)kPageSize * a->num_kv_heads * kHeadDim) * elem;
  p.scale_stride = scales && scales->page_stride > 0 ? scales->page_stride : a->num_kv_heads;
  p.hkv = a->num_kv_heads;
  p.num_pages = a->num_pages;
  p.max_pages = a->max_pages;
  p.hnd = a->kv_layout == SQA_KV_HND;
  p.budget = a->budget;
  p.recent = a->recent;
  p.sinks = a->sinks;
  const int segments = a->batch * a->num_kv_heads;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return (fp8 ? launch_evict_shape<1>(p, segments, s) : launch_evict_shape<2>(p, segments, s)) == cudaSuccess ? SQA_OK
                                                                                                            : SQA_ERR_CUDA;
}
