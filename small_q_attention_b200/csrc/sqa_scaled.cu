// sqa_scaled.cu -- attention over a block-scaled e4m3 cache, and the attention weight of
// every cached token.
//
// One CTA per (sequence, KV head) walks the sequence in tiles of 32 tokens held in
// shared memory as fp32: scores, a running maximum and sum per row, and the output
// accumulators in registers.
#include "sqa_internal.h"
#include "sqa_ptx.cuh"
#include "sqa_scaled.cuh"

namespace sqa {
namespace {

__device__ __forceinline__ void raise(unsigned int* status, unsigned int bits) {
  if (status != nullptr) atomicOr(status, bits);
}

constexpr int kTile = 32;
constexpr int kScaledThreads = 256;
constexpr int kRowStride = kHeadDim + 4;

struct ScaledSmem {
  float q[kGroup * 16][kRowStride];
  float k[kTile][kRowStride];
  float v[kTile][kRowStride];
  float s[kGroup * 16][kTile + 1];
  float m[kGroup * 16], l[kGroup * 16], alpha[kGroup * 16];
};

// kElem: 1 = e4m3 with a scale, 2 = 16-bit.
template <bool BF, int kElem>
__device__ __forceinline__ float cached(const void* cache, size_t at, float scale) {
  if constexpr (kElem == 1) {
    return unpack_e4m3x2(static_cast<const uint8_t*>(cache)[at]).x * scale;
  } else {
    return unpack2<BF>(static_cast<const uint16_t*>(cache)[at]).x;
  }
}

// Scores of tile [t0, t0 + 32) of rows `rows` into sm.s (unseen: -inf); V too for attention.
template <bool BF, int kElem, bool kWithV>
__device__ void load_tile(const ScaledParams& p, ScaledSmem& sm, int b, int h, int t0, int len, int mlen) {
  const int rows = kGroup * p.q_len;
  for (int i = threadIdx.x; i < kTile * kHeadDim; i += kScaledThreads) {
    const int t = t0 + i / kHeadDim, d = i % kHeadDim;
    float k = 0.f, v = 0.f;
    if (t < len) {
      int page = __ldg(p.block_tables + (size_t)b * p.max_pages + t / kPageSize);
      if (page < 0 || page >= p.num_pages) {
        raise(p.status, 8u);
        page = 0;
      }
      const int slot = t % kPageSize;
      const size_t at = (size_t)page * p.page_stride +
                        (p.hnd ? ((size_t)h * kPageSize + slot) : ((size_t)slot * p.hkv + h)) * kHeadDim + d;
      const size_t sc = (size_t)page * p.scale_stride + h;
      k = cached<BF, kElem>(p.k_cache, at, kElem == 1 ? p.k_scales[sc] : 1.f);
      if (kWithV) v = cached<BF, kElem>(p.v_cache, at, p.v_scales[sc]);
    }
    sm.k[i / kHeadDim][d] = k;
    if (kWithV) sm.v[i / kHeadDim][d] = v;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * kTile; i += kScaledThreads) {
    const int r = i / kTile, c = i % kTile, t = t0 + c;
    float x = 0.f;
    for (int d = 0; d < kHeadDim; ++d) x = fmaf(sm.q[r][d], sm.k[c][d], x);
    sm.s[r][c] = (t < len && t < mlen - p.q_len + (r >> 2) + 1) ? x * p.scale_log2 : -INFINITY;
  }
  __syncthreads();
}

template <bool BF>
__device__ void load_q(const ScaledParams& p, ScaledSmem& sm, int b, int h) {
  for (int i = threadIdx.x; i < kGroup * p.q_len * kHeadDim; i += kScaledThreads) {
    const int r = i / kHeadDim, d = i % kHeadDim;
    const size_t row = (size_t)(b * p.q_len + (r >> 2)) * p.hq + h * kGroup + (r & 3);
    sm.q[r][d] = unpack2<BF>(static_cast<const uint16_t*>(p.q)[row * kHeadDim + d]).x;
  }
}

template <bool BF>
__global__ void __launch_bounds__(kScaledThreads) sqa_scaled_attention_kernel(const ScaledParams p) {
  extern __shared__ uint8_t raw[];
  ScaledSmem& sm = *reinterpret_cast<ScaledSmem*>(raw);
  grid_dependency_wait();
  allow_dependent_launch();
  const int b = blockIdx.x / p.hkv, h = blockIdx.x % p.hkv;
  const int rows = kGroup * p.q_len, tid = threadIdx.x;
  const int raw_len = __ldg(p.seq_lens + b);
  const int len = min(max(raw_len, 0), p.max_pages * kPageSize);
  const int mlen = p.mask_lens ? __ldg(p.mask_lens + b) : raw_len;
  if (tid == 0) {
    if (raw_len > p.max_pages * kPageSize) raise(p.status, 2u);
    if (p.out != nullptr && raw_len < p.q_len) raise(p.status, 4u);
  }
  load_q<BF>(p, sm, b, h);
  for (int r = tid; r < rows; r += kScaledThreads) {
    sm.m[r] = -INFINITY;
    sm.l[r] = 0.f;
  }
  const int d = tid % kHeadDim, r0 = tid / kHeadDim;
  float acc[kGroup * 16 / 2];
  for (int i = 0; i < kGroup * 16 / 2; ++i) acc[i] = 0.f;
  __syncthreads();
  for (int t0 = 0; t0 < len; t0 += kTile) {
    load_tile<BF, 1, true>(p, sm, b, h, t0, len, mlen);
    if (tid < rows) {
      float m = sm.m[tid];
      for (int c = 0; c < kTile; ++c) m = fmaxf(m, sm.s[tid][c]);
      const float base = m == -INFINITY ? 0.f : m;
      float l = sm.l[tid] * ex2(sm.m[tid] - base);
      sm.alpha[tid] = ex2(sm.m[tid] - base);
      for (int c = 0; c < kTile; ++c) {
        const float e = ex2(sm.s[tid][c] - base);
        sm.s[tid][c] = e;
        l += e;
      }
      sm.m[tid] = m;
      sm.l[tid] = l;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kGroup * 16 / 2; ++i) {
      const int r = r0 + 2 * i;
      if (r < rows) {
        float a = acc[i] * sm.alpha[r];
        for (int c = 0; c < kTile; ++c)
          if (sm.s[r][c] != 0.f) a = fmaf(sm.s[r][c], sm.v[c][d], a);
        acc[i] = a;
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < kGroup * 16 / 2; ++i) {
    const int r = r0 + 2 * i;
    if (r < rows) {
      const float l = sm.l[r];
      const float o = l > 0.f || l != l ? acc[i] * p.out_scale / l : 0.f;
      const size_t row = (size_t)(b * p.q_len + (r >> 2)) * p.hq + h * kGroup + (r & 3);
      if (p.out != nullptr) static_cast<uint16_t*>(p.out)[row * kHeadDim + d] = (uint16_t)(pack2<BF>(o, 0.f) & 0xffffu);
      if (p.out_o != nullptr) p.out_o[row * kHeadDim + d] = o;
      if (p.out_lse != nullptr && d == 0)
        p.out_lse[row] = l > 0.f ? (sm.m[r] + log2f(l)) * 0.6931471805599453f : (l != l ? l : -INFINITY);
    }
  }
}

template <bool BF, int kElem>
__global__ void __launch_bounds__(kScaledThreads) sqa_weights_kernel(const ScaledParams p) {
  extern __shared__ uint8_t raw[];
  ScaledSmem& sm = *reinterpret_cast<ScaledSmem*>(raw);
  grid_dependency_wait();
  allow_dependent_launch();
  const int b = blockIdx.x / p.hkv, h = blockIdx.x % p.hkv;
  const int rows = kGroup * p.q_len, tid = threadIdx.x;
  const int raw_len = __ldg(p.seq_lens + b);
  const int len = min(max(raw_len, 0), p.max_pages * kPageSize);
  const int mlen = p.mask_lens ? __ldg(p.mask_lens + b) : raw_len;
  if (tid == 0) {
    if (raw_len > p.max_pages * kPageSize) raise(p.status, 2u);
    if (raw_len < p.q_len) raise(p.status, 4u);
  }
  load_q<BF>(p, sm, b, h);
  for (int r = tid; r < rows; r += kScaledThreads)
    sm.m[r] = p.lse[(size_t)(b * p.q_len + (r >> 2)) * p.hq + h * kGroup + (r & 3)] * 1.4426950408889634f;
  __syncthreads();
  for (int t0 = 0; t0 < len; t0 += kTile) {
    load_tile<BF, kElem, false>(p, sm, b, h, t0, len, mlen);
    const int t = t0 + tid;
    if (tid < kTile && t < len) {
      float w = 0.f;
      for (int r = 0; r < rows; ++r)
        if (sm.m[r] != -INFINITY) w += ex2(sm.s[r][tid] - sm.m[r]);
      const int page = __ldg(p.block_tables + (size_t)b * p.max_pages + t / kPageSize);
      if (page >= 0 && page < p.num_pages) {
        float* const at = p.scores + ((size_t)page * p.hkv + h) * kPageSize + t % kPageSize;
        *at = t >= raw_len - p.q_len ? w : *at + w;
      }
    }
    __syncthreads();
  }
}

cudaError_t launch(void (*kernel)(const ScaledParams), const ScaledParams& p, cudaStream_t stream) {
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(ScaledSmem));
  if (err != cudaSuccess) return err;
  kernel<<<p.batch * p.hkv, kScaledThreads, sizeof(ScaledSmem), stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_scaled_attention(const ScaledParams& p, cudaStream_t stream) {
  return launch(p.bf16 ? sqa_scaled_attention_kernel<true> : sqa_scaled_attention_kernel<false>, p, stream);
}

cudaError_t launch_weights(const ScaledParams& p, cudaStream_t stream) {
  if (p.k_scales != nullptr)
    return launch(p.bf16 ? sqa_weights_kernel<true, 1> : sqa_weights_kernel<false, 1>, p, stream);
  return launch(p.bf16 ? sqa_weights_kernel<true, 2> : sqa_weights_kernel<false, 2>, p, stream);
}

}  // namespace sqa
