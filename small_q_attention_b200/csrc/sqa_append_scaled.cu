// sqa_append_scaled.cu -- append new K/V to a block-scaled e4m3 cache.
//
// Token qi of sequence b is position t = seq_lens[b] - q_len + qi (seq_lens is the
// length after the append), in page block_tables[b, t / 16], slot t % 16, as in
// sqa_append.cu.  Per touched page and KV head, K and V apart:
//
//   need  = page_scale(max |x| over the page's finite new values)
//   scale = need                      when the page's first slot is new
//         = max(old scale, need)      otherwise
//   new values are stored as e4m3(x / scale), saturating; NaN stays NaN;
//   older tokens of the page become e4m3(q * old / scale) where the scale grew.
//
// One warp holds one page of one head of K or V: each lane owns 4 dims (8 bytes of a
// 16-bit row, 4 of an e4m3 row) of up to 16 tokens, so the maximum is one warp
// reduction over registers, every load of the page is in flight at once and each
// value is read and written once.
#include "small_q_attention.h"
#include "sqa_internal.h"
#include "sqa_ptx.cuh"
#include "sqa_scaled.cuh"

namespace sqa {
namespace {

// 64 registers: the loads of 32 pages an SM in flight (2 x 5003 tokens: 12.4 us; 13.0 with 3 blocks, 14.3 with 2,
// 20 calls each).  Back to back 14.3 us, 66% of the copy rate (floor 9.5 us).
constexpr int kBlocksPerSm = 4;

struct AppendScaledParams {
  const uint2* new_k;  // [batch, q_len, hkv, 128] 16-bit, 32 uint2 per row
  const uint2* new_v;
  uint8_t* k_cache;
  uint8_t* v_cache;
  float* k_scales;  // [num_pages, hkv], scale_stride floats from page to page
  float* v_scales;
  const int32_t* block_tables;
  const int32_t* seq_lens;
  unsigned int* status;  // may be null
  long long items;       // batch * touched * hkv * 2
  long long page_stride, scale_stride;
  int touched;  // pages that q_len tokens can touch
  int q_len, hkv, num_pages, max_pages, hnd;
};

template <bool BF>
__global__ void __launch_bounds__(256, kBlocksPerSm) sqa_cache_append_scaled_kernel(const AppendScaledParams p) {
  grid_dependency_wait();    // the previous kernel may have produced the new K/V, the cache or the tables
  allow_dependent_launch();  // what follows waits for this grid to finish
  const int lane = threadIdx.x & 31;
  unsigned int bad = 0;
  const long long stride = (long long)gridDim.x * (blockDim.x / 32);
  for (long long i = (long long)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5); i < p.items; i += stride) {
    const bool value = i & 1;
    long long r = i >> 1;
    const int h = (int)(r % p.hkv);
    r /= p.hkv;
    const int j = (int)(r % p.touched);
    const int b = (int)(r / p.touched);
    const int len = __ldg(p.seq_lens + b);
    const int t0 = len - p.q_len;
    if (len < p.q_len) {
      bad |= 4u;  // SQA_DEV_SEQ_TOO_SHORT: the whole sequence is skipped
      continue;
    }
    if (page_count(len) > p.max_pages) {
      bad |= 2u;  // SQA_DEV_SEQ_TOO_LONG: the whole sequence is skipped
      continue;
    }
    const int first = (t0 / kPageSize + j) * kPageSize;  // the page's first position
    if (first >= len) continue;
    const int page = __ldg(p.block_tables + (size_t)b * p.max_pages + first / kPageSize);
    if (page < 0 || page >= p.num_pages) {
      bad |= 8u;  // SQA_DEV_BAD_PAGE: this page is skipped
      continue;
    }
    const int n0 = max(t0 - first, 0);              // slots before n0 are older tokens
    const int n1 = min(len - first, kPageSize);     // slots from n1 on are not in use
    const uint2* src = (value ? p.new_v : p.new_k) + ((size_t)b * p.q_len * p.hkv + h) * 32 + lane;
    uint8_t* dst = (value ? p.v_cache : p.k_cache) + (size_t)page * p.page_stride +
                   (p.hnd ? (size_t)h * kPageSize * kHeadDim : (size_t)h * kHeadDim) + lane * 4;
    const size_t row = p.hnd ? kHeadDim : (size_t)p.hkv * kHeadDim;  // bytes from slot to slot
    float* const scale_at = (value ? p.v_scales : p.k_scales) + (size_t)page * p.scale_stride + h;

    uint2 x[kPageSize];
#pragma unroll
    for (int s = 0; s < kPageSize; ++s)
      x[s] = (s >= n0 && s < n1) ? __ldg(src + (size_t)(first + s - t0) * p.hkv * 32) : make_uint2(0u, 0u);
    const float was = n0 > 0 ? __ldcg(scale_at) : 0.f;
    // |x| of two 16-bit values at once, as integers (their order is that of the magnitudes); a page
    // with an infinity or NaN is looked through again for its finite values
    constexpr uint32_t kInf = BF ? 0x7f80u : 0x7c00u;
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < kPageSize; ++s) top = __vmaxu2(top, __vmaxu2(x[s].x & 0x7fff7fffu, x[s].y & 0x7fff7fffu));
    float2 m = unpack2<BF>(top);
    if ((top & 0xffffu) >= kInf || (top >> 16) >= kInf) {
      m = make_float2(0.f, 0.f);
#pragma unroll
      for (int s = 0; s < kPageSize; ++s) {
        const float2 a = unpack2<BF>(x[s].x), c = unpack2<BF>(x[s].y);
        m.x = fmaxf(m.x, fmaxf(finite_abs(a.x), finite_abs(a.y)));
        m.y = fmaxf(m.y, fmaxf(finite_abs(c.x), finite_abs(c.y)));
      }
    }
    const float amax = fmaxf(m.x, m.y);
    const float need = page_scale(warp_max(amax));
    const float scale = n0 > 0 ? fmaxf(was, need) : need;
    // Dividing by a power of two is multiplying by its reciprocal (exact; 64 IEEE divisions a lane
    // made a prompt's append four times as long).  Only an old scale that another quantiser
    // chose can be anything else.
    const bool power = (__float_as_uint(scale) & 0x7fffffu) == 0u;
    const float inv = 1.f / scale;
    if (n0 > 0 && scale > was) {  // the older tokens follow the page's new scale, a power of two
      uint32_t q[kPageSize];
#pragma unroll
      for (int s = 0; s < kPageSize; ++s) q[s] = s < n0 ? __ldcg(reinterpret_cast<const uint32_t*>(dst + s * row)) : 0u;
#pragma unroll
      for (int s = 0; s < kPageSize; ++s) {
        if (s < n0) {
          const float2 a = unpack_e4m3x2(q[s]), c = unpack_e4m3x2(q[s] >> 16);
          *reinterpret_cast<uint32_t*>(dst + s * row) =
              pack_e4m3x4(a.x * was * inv, a.y * was * inv, c.x * was * inv, c.y * was * inv);
        }
      }
    }
    if (!BF && power && inv >= 6.103515625e-05f && inv <= 16384.f) {
      // fp16: the product in fp16, exact but for results below 2^-14, which are zero in e4m3 as well
      const __half2 f = __float2half2_rn(inv);
#pragma unroll
      for (int s = 0; s < kPageSize; ++s) {
        if (s >= n0 && s < n1) {
          const __half2 a = *reinterpret_cast<const __half2*>(&x[s].x), c = *reinterpret_cast<const __half2*>(&x[s].y);
          *reinterpret_cast<uint32_t*>(dst + s * row) = e4m3x2_of_half2(__hmul2(a, f)) | (e4m3x2_of_half2(__hmul2(c, f)) << 16);
        }
      }
    } else if (power) {
#pragma unroll
      for (int s = 0; s < kPageSize; ++s) {
        if (s >= n0 && s < n1) {
          const float2 a = unpack2<BF>(x[s].x), c = unpack2<BF>(x[s].y);
          *reinterpret_cast<uint32_t*>(dst + s * row) = pack_e4m3x4(a.x * inv, a.y * inv, c.x * inv, c.y * inv);
        }
      }
    } else {
#pragma unroll 1
      for (int s = n0; s < n1; ++s) {  // not unrolled: x is read again
        const uint2 y = __ldg(src + (size_t)(first + s - t0) * p.hkv * 32);
        const float2 a = unpack2<BF>(y.x), c = unpack2<BF>(y.y);
        *reinterpret_cast<uint32_t*>(dst + s * row) =
            pack_e4m3x4(__fdiv_rn(a.x, scale), __fdiv_rn(a.y, scale), __fdiv_rn(c.x, scale), __fdiv_rn(c.y, scale));
      }
    }
    if (lane == 0) *scale_at = scale;
  }
  if (bad && lane == 0 && p.status != nullptr) atomicOr(p.status, bad);
}

}  // namespace
}  // namespace sqa

using namespace sqa;

extern "C" SQA_API int sqa_cache_append_scaled(const sqa_append_args* a, const sqa_scales* scales, int32_t new_dtype,
                                               void* stream) {
  if (a == nullptr || scales == nullptr) return SQA_ERR_INVALID_ARGUMENT;
  if (a->head_dim != kHeadDim || a->page_size != kPageSize) return SQA_ERR_UNSUPPORTED;
  if (a->batch < 0 || a->q_len <= 0 || a->num_kv_heads <= 0 || a->num_pages <= 0 || a->max_pages <= 0)
    return SQA_ERR_INVALID_ARGUMENT;
  if (a->kv_layout != SQA_KV_NHD && a->kv_layout != SQA_KV_HND) return SQA_ERR_UNSUPPORTED;
  if (a->kv_dtype != SQA_KV_FP8_E4M3) return SQA_ERR_UNSUPPORTED;
  if (new_dtype != SQA_DTYPE_F16 && new_dtype != SQA_DTYPE_BF16) return SQA_ERR_UNSUPPORTED;
  if (a->page_stride < 0 || (a->page_stride > 0 && (a->page_stride < (int64_t)kPageSize * a->num_kv_heads * kHeadDim ||
                                                    a->page_stride % 16 != 0)))
    return SQA_ERR_INVALID_ARGUMENT;
  if (scales->page_stride < 0 || (scales->page_stride > 0 && scales->page_stride < a->num_kv_heads))
    return SQA_ERR_INVALID_ARGUMENT;
  if (a->max_pages > (1 << 26)) return SQA_ERR_UNSUPPORTED;  // positions are 32-bit
  if (a->batch == 0) return SQA_OK;
  if (!a->new_keys || !a->new_values || !a->key_cache || !a->value_cache || !a->block_tables || !a->seq_lens ||
      !scales->key || !scales->value)
    return SQA_ERR_INVALID_ARGUMENT;
  const uintptr_t wide = reinterpret_cast<uintptr_t>(a->new_keys) | reinterpret_cast<uintptr_t>(a->new_values) |
                         reinterpret_cast<uintptr_t>(a->key_cache) | reinterpret_cast<uintptr_t>(a->value_cache);
  const uintptr_t narrow = reinterpret_cast<uintptr_t>(a->block_tables) | reinterpret_cast<uintptr_t>(a->seq_lens) |
                           reinterpret_cast<uintptr_t>(a->status) | reinterpret_cast<uintptr_t>(scales->key) |
                           reinterpret_cast<uintptr_t>(scales->value);
  if ((wide & 15u) || (narrow & 3u)) return SQA_ERR_INVALID_ARGUMENT;

  AppendScaledParams p;
  p.new_k = static_cast<const uint2*>(a->new_keys);
  p.new_v = static_cast<const uint2*>(a->new_values);
  p.k_cache = static_cast<uint8_t*>(a->key_cache);
  p.v_cache = static_cast<uint8_t*>(a->value_cache);
  p.k_scales = scales->key;
  p.v_scales = scales->value;
  p.block_tables = a->block_tables;
  p.seq_lens = a->seq_lens;
  p.status = a->status;
  p.touched = (int)(((int64_t)a->q_len + kPageSize - 2) / kPageSize + 1);
  if (p.touched > a->max_pages) p.touched = a->max_pages;
  p.items = (long long)a->batch * p.touched * a->num_kv_heads * 2;
  p.q_len = a->q_len;
  p.hkv = a->num_kv_heads;
  p.num_pages = a->num_pages;
  p.max_pages = a->max_pages;
  p.hnd = a->kv_layout == SQA_KV_HND;
  p.page_stride = a->page_stride > 0 ? a->page_stride : (int64_t)kPageSize * a->num_kv_heads * kHeadDim;
  p.scale_stride = scales->page_stride > 0 ? scales->page_stride : a->num_kv_heads;

  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return SQA_ERR_CUDA;
  long long blocks = (p.items + 7) / 8;
  if (blocks > (long long)sms * 8) blocks = (long long)sms * 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(256);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = new_dtype == SQA_DTYPE_BF16
                              ? cudaLaunchKernelEx(&cfg, sqa_cache_append_scaled_kernel<true>, p)
                              : cudaLaunchKernelEx(&cfg, sqa_cache_append_scaled_kernel<false>, p);
  if (err != cudaSuccess) return SQA_ERR_CUDA;
  return cudaGetLastError() == cudaSuccess ? SQA_OK : SQA_ERR_CUDA;
}
