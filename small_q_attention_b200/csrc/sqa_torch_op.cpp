// sqa_torch_op.cpp -- the operator as a torch extension over the C ABI.
//
// Two doors into the same code:
// * TORCH_LIBRARY(sqa_b200): torch.ops.sqa_b200.small_q_attention /
//   small_q_attention_partial / small_q_attention_scaled, with CUDA and Meta kernels, so torch.compile and
//   fake-tensor tracing see a real operator instead of an opaque Python call;
// * a pybind11 module (_sqa_torch.forward / forward_partial) that the Python
//   entry small_q_attention() calls directly: the contract checks, argument
//   packing, workspace lookup and both launches run here in C++, on torch's
//   current stream, in a few microseconds of host time.
//
// The checks and their exception types restate the upstream Python wrapper's
// contract (src/small_q_attention/cuda.py:197-211: ValueError for a tensor
// that is not on CUDA, not contiguous, of the wrong dtype or outside the shape
// contract); the launch is sqa_forward (include/small_q_attention.h), which
// replaces small_q_attention_v3 (csrc/small_q_attention_ext.cu:1132-1210).
// Nothing here computes: every kernel lives in libsqa_b200.so.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>
#include <torch/library.h>

#include <memory>
#include <mutex>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/small_q_attention.h"

namespace {

constexpr int64_t kHeadDim = SQA_HEAD_DIM;
constexpr int64_t kPage = SQA_PAGE_SIZE;
constexpr int64_t kGroup = SQA_GQA_GROUP;
constexpr int64_t kMaxQ = SQA_MAX_Q_LEN;

// Elements from one page to the next (0 = contiguous caches); the caches may be
// views of a bigger pool: packed within a page, one 16-byte aligned page
// stride shared by K and V.
int64_t cache_page_stride(const at::Tensor& k, const at::Tensor& v) {
  TORCH_CHECK_VALUE(k.dim() == 4, "key_cache must be 4-D");
  if (k.is_contiguous() && v.is_contiguous()) return 0;
  const auto st = k.strides();
  const int64_t inner = k.size(1) * k.size(2) * k.size(3);
  const int64_t align = 16 / k.element_size();
  const bool packed = st[1] == k.size(2) * k.size(3) && st[2] == k.size(3) && st[3] == 1;
  TORCH_CHECK_VALUE(v.strides() == st && packed && st[0] >= inner && st[0] % align == 0,
                    "key_cache / value_cache must be packed within a page, with one page stride "
                    "(16-byte aligned) shared by K and V");
  return st[0];
}

void check_inputs(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& bt,
                  const at::Tensor& sl, int64_t page_size, const c10::optional<at::Tensor>& mask_lens,
                  int64_t kv_layout) {
  const at::Tensor* all[6] = {&q, &k, &v, &bt, &sl, mask_lens.has_value() ? &*mask_lens : nullptr};
  const int n = mask_lens.has_value() ? 6 : 5;
  for (int i = 0; i < n; ++i) TORCH_CHECK_VALUE(all[i]->defined(), "all inputs must be CUDA tensors");
  TORCH_CHECK_VALUE(q.is_cuda(), "all inputs must be CUDA tensors");
  const auto dev = q.device();
  for (int i = 0; i < n; ++i) {
    TORCH_CHECK_VALUE(all[i]->device() == dev, "all inputs must be CUDA tensors on the same device");
    if (i != 1 && i != 2) TORCH_CHECK_VALUE(all[i]->is_contiguous(), "all inputs must be contiguous");
  }
  cache_page_stride(k, v);
  const auto qd = q.scalar_type(), kd = k.scalar_type();
  TORCH_CHECK_VALUE((qd == at::kHalf || qd == at::kBFloat16) && v.scalar_type() == kd &&
                        (kd == qd || kd == at::kFloat8_e4m3fn),
                    "the kernel requires FP16 (or BF16) Q/K/V of one type, or FP16/BF16 Q with FP8-E4M3 K/V");
  for (int i = 3; i < n; ++i)
    TORCH_CHECK_VALUE(all[i]->scalar_type() == at::kInt, "block_tables, seq_lens and mask_lens must be int32");
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4, "query and key_cache must be 4-D");
  TORCH_CHECK_VALUE(v.sizes() == k.sizes(), "value_cache shape mismatch");
  TORCH_CHECK_VALUE(kv_layout == SQA_KV_NHD || kv_layout == SQA_KV_HND,
                    "kv_layout must be \"NHD\" ([pages, 16, Hkv, 128]) or \"HND\" ([pages, Hkv, 16, 128])");
  const int64_t batch = q.size(0), q_len = q.size(1), hq = q.size(2), head_dim = q.size(3);
  const bool hnd = kv_layout == SQA_KV_HND;
  const int64_t hkv = hnd ? k.size(1) : k.size(2);
  const int64_t cache_page = hnd ? k.size(2) : k.size(1);
  TORCH_CHECK_VALUE(q_len >= 1 && q_len <= kMaxQ, "q_len must be in [1, ", kMaxQ, "]");
  TORCH_CHECK_VALUE(head_dim == kHeadDim && k.size(3) == kHeadDim, "the kernel supports head_dim 128");
  TORCH_CHECK_VALUE(hkv > 0 && hq % hkv == 0 && hq / hkv == kGroup,
                    "the kernel requires a GQA group size of exactly 4 (Hq/Hkv = 32/8)");
  TORCH_CHECK_VALUE(page_size == cache_page && cache_page == kPage,
                    "page_size must be 16 and match the cache's page dimension");
  TORCH_CHECK_VALUE(bt.dim() == 2 && bt.size(0) == batch && sl.numel() == batch,
                    "invalid metadata: block_tables must be [batch, max_pages], seq_lens [batch]");
  TORCH_CHECK_VALUE(!mask_lens.has_value() || mask_lens->numel() == batch,
                    "mask_lens must have one entry per sequence");
  TORCH_CHECK_VALUE(k.size(0) > 0 && bt.size(1) > 0, "empty KV cache is not supported");
}

sqa_args fill_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& bt,
                   const at::Tensor& sl, const c10::optional<at::Tensor>& mask_lens, int64_t max_seq_len,
                   int64_t num_ctas, int64_t min_pages_per_cta, int64_t kernel, int64_t kv_layout, double sm_scale,
                   double out_scale, int64_t min_seq_len = 0, int64_t cluster = 0) {
  sqa_args a = {};
  const bool hnd = kv_layout == SQA_KV_HND;
  a.query = q.data_ptr();
  a.key_cache = k.data_ptr();
  a.value_cache = v.data_ptr();
  a.block_tables = bt.data_ptr<int32_t>();
  a.seq_lens = sl.data_ptr<int32_t>();
  a.mask_lens = mask_lens.has_value() ? mask_lens->data_ptr<int32_t>() : nullptr;
  a.batch = (int32_t)q.size(0);
  a.q_len = (int32_t)q.size(1);
  a.num_q_heads = (int32_t)q.size(2);
  a.num_kv_heads = (int32_t)(hnd ? k.size(1) : k.size(2));
  a.head_dim = (int32_t)q.size(3);
  a.page_size = (int32_t)(hnd ? k.size(2) : k.size(1));
  a.num_pages = (int32_t)k.size(0);
  a.max_pages = (int32_t)bt.size(1);
  a.max_seq_len = (int32_t)max_seq_len;
  a.num_ctas = (int32_t)num_ctas;
  a.min_pages_per_cta = (int32_t)min_pages_per_cta;
  a.kernel = (int32_t)kernel;
  a.dtype = q.scalar_type() == at::kBFloat16 ? SQA_DTYPE_BF16 : SQA_DTYPE_F16;
  a.kv_layout = (int32_t)kv_layout;
  a.sm_scale = (float)sm_scale;
  a.out_scale = (float)out_scale;
  a.page_stride = cache_page_stride(k, v);
  a.kv_dtype = k.scalar_type() == at::kFloat8_e4m3fn ? SQA_KV_FP8_E4M3 : SQA_KV_SAME;
  a.min_seq_len = (int32_t)min_seq_len;
  a.cluster = (int32_t)cluster;
  return a;
}

void check_status(int code, const char* what) {
  if (code == SQA_OK) return;
  const std::string msg = std::string(what) + ": " + sqa_status_string(code) + " (status " + std::to_string(code) + ")";
  TORCH_CHECK_VALUE(code != SQA_ERR_INVALID_ARGUMENT && code != SQA_ERR_UNSUPPORTED, msg);
  TORCH_CHECK(false, msg);
}

// The memory of one call.  A registered operator runs without Python's lock, so calls from two host threads on
// one stream meet here: the launches of a call that use a shared workspace hold `turn`, or the
// other call's kernels would come between its split and its merge.
struct CallMemory {
  at::Tensor ws;
  std::shared_ptr<std::mutex> turn;  // null: the call's own memory, or the caller's
  std::unique_lock<std::mutex> hold() const { return turn ? std::unique_lock<std::mutex>(*turn) : std::unique_lock<std::mutex>(); }
};

// One workspace per (device, stream), grown on demand; the status word of a
// new one starts zeroed.  (A caller's explicit workspace is used as given.)
struct WsEntry {
  int device;
  cudaStream_t stream;
  CallMemory mem;
};
std::mutex g_ws_mu;
std::vector<WsEntry> g_ws;

CallMemory workspace_for(const sqa_args& a, const at::Device& dev, cudaStream_t stream,
                         const c10::optional<at::Tensor>& workspace) {
  if (workspace.has_value()) {
    const at::Tensor& w = *workspace;
    TORCH_CHECK_VALUE(w.device() == dev && w.is_contiguous(),
                      "workspace must be a contiguous tensor on the query's device");
    return {w, nullptr};
  }
  int st = SQA_OK;
  const size_t need = sqa_workspace_bytes(&a, dev.index(), &st);
  check_status(st, "sqa_workspace_bytes");
  std::lock_guard<std::mutex> lock(g_ws_mu);
  for (auto& e : g_ws) {
    if (e.device == dev.index() && e.stream == stream) {
      if ((size_t)e.mem.ws.numel() < need) e.mem.ws = at::zeros({(int64_t)std::max<size_t>(need, 1 << 20)},
                                                                at::TensorOptions().dtype(at::kByte).device(dev));
      return e.mem;
    }
  }
  g_ws.push_back(WsEntry{dev.index(), stream,
                         {at::zeros({(int64_t)std::max<size_t>(need, 1 << 20)}, at::TensorOptions().dtype(at::kByte).device(dev)),
                          std::make_shared<std::mutex>()}});
  return g_ws.back().mem;
}

// check=True: synchronise and raise what the upstream CPU reference raises
// for bad metadata (reference.py:52-53; index_select on a bad page id).
void raise_device_bits(void* ws, cudaStream_t stream) {
  uint32_t bits = 0;
  const int code = sqa_read_device_status(ws, &bits, 1, stream);
  if (code != SQA_OK && code != SQA_ERR_DEVICE) check_status(code, "sqa_read_device_status");
  TORCH_CHECK_VALUE(!(bits & SQA_DEV_SEQ_TOO_SHORT), "seq_lens must be at least q_len for MTP attention");
  TORCH_CHECK_VALUE(!(bits & SQA_DEV_SEQ_TOO_LONG), "seq_lens exceeds page_size * block_tables.shape[1]");
  TORCH_CHECK_INDEX(!(bits & SQA_DEV_BAD_PAGE), "block_tables holds a page id outside the cache");
  TORCH_CHECK(!(bits & SQA_DEV_TIMEOUT), "a bounded device wait timed out; the output is not valid");
}

void launch(sqa_args& a, const at::Tensor& q, const c10::optional<at::Tensor>& workspace, bool check) {
  const at::Device dev = q.device();
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != dev.index()) guard.set_index(dev.index());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  const CallMemory mem = workspace_for(a, dev, stream, workspace);
  const auto turn = mem.hold();
  void* const ws = mem.ws.data_ptr();
  const int code = sqa_forward(&a, ws, (size_t)mem.ws.numel() * mem.ws.element_size(), stream);
  if (code == SQA_ERR_WORKSPACE_TOO_SMALL && workspace.has_value()) {
    int st = SQA_OK;
    TORCH_CHECK_VALUE(false, "workspace too small: need ", sqa_workspace_bytes(&a, dev.index(), &st), " bytes");
  }
  check_status(code, "sqa_forward");
  if (check) raise_device_bits(ws, stream);
}

at::Tensor forward(const at::Tensor& query, const at::Tensor& key_cache, const at::Tensor& value_cache,
                   const at::Tensor& block_tables, const at::Tensor& seq_lens, int64_t page_size, int64_t max_seq_len,
                   const c10::optional<at::Tensor>& out, const c10::optional<at::Tensor>& workspace, int64_t num_ctas,
                   int64_t min_pages_per_cta, int64_t kernel, bool check, int64_t kv_layout, double sm_scale,
                   double out_scale, int64_t min_seq_len, int64_t cluster) {
  check_inputs(query, key_cache, value_cache, block_tables, seq_lens, page_size, c10::nullopt, kv_layout);
  at::Tensor o;
  if (out.has_value()) {
    o = *out;
    TORCH_CHECK_VALUE(o.sizes() == query.sizes() && o.scalar_type() == query.scalar_type() && o.is_contiguous() &&
                          o.device() == query.device(),
                      "out must be a contiguous tensor shaped and typed like query");
  } else {
    o = at::empty_like(query);
  }
  sqa_args a = fill_args(query, key_cache, value_cache, block_tables, seq_lens, c10::nullopt, max_seq_len, num_ctas,
                         min_pages_per_cta, kernel, kv_layout, sm_scale, out_scale, min_seq_len, cluster);
  a.out = o.data_ptr();
  launch(a, query, workspace, check);
  return o;
}

std::tuple<at::Tensor, at::Tensor> forward_partial(
    const at::Tensor& query, const at::Tensor& key_cache, const at::Tensor& value_cache,
    const at::Tensor& block_tables, const at::Tensor& seq_lens, int64_t page_size,
    const c10::optional<at::Tensor>& mask_lens, int64_t max_seq_len, const c10::optional<at::Tensor>& out,
    const c10::optional<at::Tensor>& out_lse, const c10::optional<at::Tensor>& workspace, int64_t num_ctas,
    int64_t min_pages_per_cta, int64_t kernel, bool check, int64_t kv_layout, double sm_scale, double out_scale,
    int64_t min_seq_len, int64_t cluster) {
  check_inputs(query, key_cache, value_cache, block_tables, seq_lens, page_size, mask_lens, kv_layout);
  const auto f32 = query.options().dtype(at::kFloat);
  at::Tensor o = out.has_value() ? *out : at::empty(query.sizes(), f32);
  at::Tensor l = out_lse.has_value() ? *out_lse : at::empty(query.sizes().slice(0, 3), f32);
  TORCH_CHECK_VALUE(o.scalar_type() == at::kFloat && o.sizes() == query.sizes() && o.is_contiguous() &&
                        o.device() == query.device(),
                    "out must be a contiguous fp32 tensor shaped like query");
  TORCH_CHECK_VALUE(l.scalar_type() == at::kFloat && l.sizes() == query.sizes().slice(0, 3) && l.is_contiguous() &&
                        l.device() == query.device(),
                    "out_lse must be a contiguous fp32 tensor [batch, q_len, Hq]");
  sqa_args a = fill_args(query, key_cache, value_cache, block_tables, seq_lens, mask_lens, max_seq_len, num_ctas,
                         min_pages_per_cta, kernel, kv_layout, sm_scale, out_scale, min_seq_len, cluster);
  a.out_partial = o.data_ptr<float>();
  a.out_lse = l.data_ptr<float>();
  launch(a, query, workspace, check);
  return {o, l};
}

// ---- the block-scaled e4m3 cache and eviction by attention weight

// Scales [num_pages, Hkv] fp32, K and V alike; rows may be further apart than Hkv.
sqa_scales fill_scales(const at::Tensor& k, const at::Tensor& v, const at::Tensor& cache, int64_t hkv) {
  for (const at::Tensor* t : {&k, &v}) {
    TORCH_CHECK_VALUE(t->defined() && t->device() == cache.device(), "all inputs must be CUDA tensors on the same device");
    TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(0) == cache.size(0) && t->size(1) == hkv,
                      "key_scales / value_scales must be fp32 [num_pages, Hkv]");
    TORCH_CHECK_VALUE((hkv == 1 || t->stride(1) == 1) && (t->size(0) == 1 || t->stride(0) >= hkv) &&
                          (t->size(0) == 1 || t->stride(0) == k.stride(0)),
                      "key_scales / value_scales must be packed over the heads, with one page stride shared by both");
  }
  return sqa_scales{k.data_ptr<float>(), v.data_ptr<float>(), k.size(0) == 1 ? hkv : k.stride(0)};
}

// Memory of a call whose first word is its status word.  Eagerly one tensor per
// (device, stream, use), grown on demand and zeroed once.  Under stream capture a
// fresh one from the capture's own pool, its status word zeroed by the graph: two
// captured graphs never share it, whatever streams they are replayed on.
enum Use { kUseAttention, kUseAppend, kUseWeights, kUseEvict };
struct UseEntry {
  int device;
  cudaStream_t stream;
  Use use;
  CallMemory mem;
};
std::mutex g_use_mu;
std::vector<UseEntry> g_use;

CallMemory memory_for(Use use, size_t need, const at::Device& dev, cudaStream_t stream) {
  const auto bytes = at::TensorOptions().dtype(at::kByte).device(dev);
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  TORCH_CHECK(cudaStreamIsCapturing(stream, &cs) == cudaSuccess, "cudaStreamIsCapturing failed");
  if (cs != cudaStreamCaptureStatusNone) {
    at::Tensor ws = at::empty({(int64_t)need}, bytes);
    check_status(sqa_workspace_init(ws.data_ptr(), std::min<size_t>(need, 256), stream), "sqa_workspace_init");
    return {ws, nullptr};
  }
  std::lock_guard<std::mutex> lock(g_use_mu);
  for (auto& e : g_use) {
    if (e.device == dev.index() && e.stream == stream && e.use == use) {
      if ((size_t)e.mem.ws.numel() < need) e.mem.ws = at::zeros({(int64_t)need}, bytes);
      return e.mem;
    }
  }
  g_use.push_back(UseEntry{dev.index(), stream, use, {at::zeros({(int64_t)need}, bytes), std::make_shared<std::mutex>()}});
  return g_use.back().mem;
}

// check=True reports the bits of this call alone: earlier unchecked calls on the
// stream may have left theirs in the word.
void clear_status(const at::Tensor& ws, cudaStream_t stream) {
  check_status(sqa_workspace_init(ws.data_ptr(), std::min<size_t>((size_t)ws.numel() * ws.element_size(), 256), stream),
               "sqa_workspace_init");
}

cudaStream_t on_device(c10::cuda::OptionalCUDAGuard& guard, const at::Device& dev) {
  if (c10::cuda::current_device() != dev.index()) guard.set_index(dev.index());
  return at::cuda::getCurrentCUDAStream(dev.index()).stream();
}

std::tuple<at::Tensor, c10::optional<at::Tensor>> forward_scaled(
    const at::Tensor& query, const at::Tensor& key_cache, const at::Tensor& value_cache, const at::Tensor& key_scales,
    const at::Tensor& value_scales, const at::Tensor& block_tables, const at::Tensor& seq_lens, int64_t page_size,
    const c10::optional<at::Tensor>& mask_lens, int64_t max_seq_len, const c10::optional<at::Tensor>& out,
    const c10::optional<at::Tensor>& out_lse, bool return_lse, const c10::optional<at::Tensor>& workspace,
    int64_t num_ctas, bool check, int64_t kv_layout, double sm_scale, double out_scale, int64_t min_seq_len,
    int64_t cluster) {
  check_inputs(query, key_cache, value_cache, block_tables, seq_lens, page_size, mask_lens, kv_layout);
  TORCH_CHECK_VALUE(key_cache.scalar_type() == at::kFloat8_e4m3fn, "a block-scaled cache is FP8-E4M3");
  sqa_args a = fill_args(query, key_cache, value_cache, block_tables, seq_lens, mask_lens, max_seq_len, num_ctas, 0, 0,
                         kv_layout, sm_scale, out_scale, min_seq_len, cluster);
  TORCH_CHECK_VALUE(cluster == 0 || cluster == 1, "cluster must be 0 or 1 for a block-scaled cache");
  const sqa_scales scales = fill_scales(key_scales, value_scales, key_cache, a.num_kv_heads);
  const at::Tensor o = out.has_value() ? *out : at::empty_like(query);
  TORCH_CHECK_VALUE(o.sizes() == query.sizes() && o.is_contiguous() && o.device() == query.device() &&
                        (o.scalar_type() == query.scalar_type() || o.scalar_type() == at::kFloat),
                    "out must be a contiguous tensor shaped like query, of its type or fp32");
  const bool f32 = o.scalar_type() == at::kFloat;
  c10::optional<at::Tensor> l = out_lse;
  if (!l.has_value() && (return_lse || f32))
    l = at::empty(query.sizes().slice(0, 3), query.options().dtype(at::kFloat));
  TORCH_CHECK_VALUE(!l.has_value() || (l->scalar_type() == at::kFloat && l->sizes() == query.sizes().slice(0, 3) &&
                                       l->is_contiguous() && l->device() == query.device()),
                    "out_lse must be a contiguous fp32 tensor [batch, q_len, Hq]");
  if (f32) a.out_partial = o.data_ptr<float>();
  else a.out = o.data_ptr();
  a.out_lse = l.has_value() ? l->data_ptr<float>() : nullptr;
  const at::Device dev = query.device();
  c10::cuda::OptionalCUDAGuard guard;
  const cudaStream_t stream = on_device(guard, dev);
  int st = SQA_OK;
  const size_t need = sqa_scaled_workspace_bytes(&a, dev.index(), &st);
  check_status(st, "sqa_scaled_workspace_bytes");
  TORCH_CHECK_VALUE(!workspace.has_value() || (workspace->device() == dev && workspace->is_contiguous()),
                    "workspace must be a contiguous tensor on the query's device");
  const CallMemory mem = workspace.has_value() ? CallMemory{*workspace, nullptr} : memory_for(kUseAttention, need, dev, stream);
  const at::Tensor& ws = mem.ws;
  const size_t have = (size_t)ws.numel() * ws.element_size();
  TORCH_CHECK_VALUE(have >= need, "workspace too small: need ", need, " bytes");
  const auto turn = mem.hold();
  if (check) clear_status(ws, stream);
  check_status(sqa_forward_scaled(&a, &scales, ws.data_ptr(), have, stream), "sqa_forward_scaled");
  if (check) raise_device_bits(ws.data_ptr(), stream);
  return {o, return_lse ? l : c10::nullopt};
}

void accumulate_weights(const at::Tensor& query, const at::Tensor& key_cache, const c10::optional<at::Tensor>& key_scales,
                        const at::Tensor& block_tables, const at::Tensor& seq_lens, const at::Tensor& lse,
                        const at::Tensor& scores, int64_t page_size, const c10::optional<at::Tensor>& mask_lens,
                        int64_t max_seq_len, int64_t num_ctas, bool check, int64_t kv_layout, double sm_scale,
                        int64_t min_seq_len) {
  check_inputs(query, key_cache, key_cache, block_tables, seq_lens, page_size, mask_lens, kv_layout);
  const sqa_args a = fill_args(query, key_cache, key_cache, block_tables, seq_lens, mask_lens, max_seq_len, num_ctas, 0,
                               0, kv_layout, sm_scale, 1.0, min_seq_len, 0);
  const bool fp8 = key_cache.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK_VALUE(fp8 == key_scales.has_value(), "key_scales belong to an FP8-E4M3 cache, and to no other");
  sqa_scales scales = {};
  if (fp8) scales = fill_scales(*key_scales, *key_scales, key_cache, a.num_kv_heads);
  const at::Device dev = query.device();
  TORCH_CHECK_VALUE(lse.device() == dev && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
                        lse.sizes() == query.sizes().slice(0, 3),
                    "lse must be a contiguous fp32 tensor [batch, q_len, Hq]");
  TORCH_CHECK_VALUE(scores.device() == dev && scores.scalar_type() == at::kFloat && scores.is_contiguous() &&
                        scores.sizes() == at::IntArrayRef({key_cache.size(0), (int64_t)a.num_kv_heads, kPage}),
                    "scores must be a contiguous fp32 tensor [num_pages, Hkv, 16]");
  c10::cuda::OptionalCUDAGuard guard;
  const cudaStream_t stream = on_device(guard, dev);
  const CallMemory mem = memory_for(kUseWeights, 256, dev, stream);
  const auto turn = mem.hold();
  const at::Tensor& word = mem.ws;
  if (check) clear_status(word, stream);
  check_status(sqa_accumulate_weights(&a, lse.data_ptr<float>(), fp8 ? &scales : nullptr, scores.data_ptr<float>(),
                                      static_cast<uint32_t*>(word.data_ptr()), stream),
               "sqa_accumulate_weights");
  if (check) raise_device_bits(word.data_ptr(), stream);
}

void append_scaled(const at::Tensor& new_keys, const at::Tensor& new_values, const at::Tensor& key_cache,
                   const at::Tensor& value_cache, const at::Tensor& key_scales, const at::Tensor& value_scales,
                   const at::Tensor& block_tables, const at::Tensor& seq_lens, bool check, int64_t kv_layout) {
  TORCH_CHECK_VALUE(key_cache.is_cuda(), "all inputs must be CUDA tensors");
  const at::Device dev = key_cache.device();
  for (const at::Tensor* t : {&new_keys, &new_values, &value_cache, &block_tables, &seq_lens})
    TORCH_CHECK_VALUE(t->device() == dev, "all inputs must be CUDA tensors on the same device");
  for (const at::Tensor* t : {&new_keys, &new_values, &block_tables, &seq_lens})
    TORCH_CHECK_VALUE(t->is_contiguous(), "all inputs must be contiguous");
  const auto nt = new_keys.scalar_type();
  TORCH_CHECK_VALUE((nt == at::kHalf || nt == at::kBFloat16) && new_values.scalar_type() == nt,
                    "new K/V must be FP16 or BF16, both of one type");
  TORCH_CHECK_VALUE(key_cache.scalar_type() == at::kFloat8_e4m3fn && value_cache.scalar_type() == at::kFloat8_e4m3fn,
                    "a block-scaled cache is FP8-E4M3");
  TORCH_CHECK_VALUE(block_tables.scalar_type() == at::kInt && seq_lens.scalar_type() == at::kInt,
                    "block_tables and seq_lens must be int32");
  TORCH_CHECK_VALUE(new_keys.dim() == 4 && new_values.sizes() == new_keys.sizes(),
                    "new_keys / new_values must be [batch, q_len, Hkv, 128]");
  TORCH_CHECK_VALUE(key_cache.dim() == 4 && value_cache.sizes() == key_cache.sizes(),
                    "key_cache / value_cache must be 4-D and of one shape");
  const bool hnd = kv_layout == SQA_KV_HND;
  const int64_t batch = new_keys.size(0), q_len = new_keys.size(1), hkv = new_keys.size(2);
  TORCH_CHECK_VALUE(new_keys.size(3) == kHeadDim && key_cache.size(3) == kHeadDim, "the kernel supports head_dim 128");
  TORCH_CHECK_VALUE(key_cache.size(hnd ? 2 : 1) == kPage, "page_size must be 16");
  TORCH_CHECK_VALUE(hkv > 0 && key_cache.size(hnd ? 1 : 2) == hkv,
                    "new K/V and the caches disagree on the number of KV heads");
  TORCH_CHECK_VALUE(q_len >= 1, "q_len must be at least 1");
  TORCH_CHECK_VALUE(block_tables.dim() == 2 && block_tables.size(0) == batch && seq_lens.numel() == batch,
                    "invalid metadata: block_tables must be [batch, max_pages], seq_lens [batch]");
  TORCH_CHECK_VALUE(key_cache.size(0) > 0 && block_tables.size(1) > 0, "empty KV cache is not supported");
  const sqa_scales scales = fill_scales(key_scales, value_scales, key_cache, hkv);
  const int64_t page_stride = cache_page_stride(key_cache, value_cache);
  if (batch == 0) return;
  c10::cuda::OptionalCUDAGuard guard;
  const cudaStream_t stream = on_device(guard, dev);
  const CallMemory mem = memory_for(kUseAppend, 256, dev, stream);
  const auto turn = mem.hold();
  const at::Tensor& word = mem.ws;
  sqa_append_args a = {};
  a.new_keys = new_keys.data_ptr();
  a.new_values = new_values.data_ptr();
  a.key_cache = key_cache.data_ptr();
  a.value_cache = value_cache.data_ptr();
  a.block_tables = block_tables.data_ptr<int32_t>();
  a.seq_lens = seq_lens.data_ptr<int32_t>();
  a.status = static_cast<uint32_t*>(word.data_ptr());
  a.batch = (int32_t)batch;
  a.q_len = (int32_t)q_len;
  a.num_kv_heads = (int32_t)hkv;
  a.head_dim = (int32_t)kHeadDim;
  a.page_size = (int32_t)kPage;
  a.num_pages = (int32_t)key_cache.size(0);
  a.max_pages = (int32_t)block_tables.size(1);
  a.kv_layout = (int32_t)kv_layout;
  a.page_stride = page_stride;
  a.kv_dtype = SQA_KV_FP8_E4M3;
  if (check) clear_status(word, stream);
  check_status(sqa_cache_append_scaled(&a, &scales, nt == at::kBFloat16 ? SQA_DTYPE_BF16 : SQA_DTYPE_F16, stream),
               "sqa_cache_append_scaled");
  if (check) raise_device_bits(word.data_ptr(), stream);
}

std::tuple<at::Tensor, at::Tensor> cache_evict(const at::Tensor& key_cache, const at::Tensor& value_cache,
                                               const at::Tensor& scores, const at::Tensor& block_tables,
                                               const at::Tensor& seq_lens, int64_t budget, int64_t recent, int64_t sinks,
                                               const c10::optional<at::Tensor>& key_scales,
                                               const c10::optional<at::Tensor>& value_scales,
                                               const c10::optional<at::Tensor>& new_lens,
                                               const c10::optional<at::Tensor>& kept, bool check, int64_t kv_layout) {
  TORCH_CHECK_VALUE(key_cache.is_cuda(), "all inputs must be CUDA tensors");
  const at::Device dev = key_cache.device();
  for (const at::Tensor* t : {&value_cache, &scores, &block_tables, &seq_lens})
    TORCH_CHECK_VALUE(t->device() == dev, "all inputs must be CUDA tensors on the same device");
  for (const at::Tensor* t : {&scores, &block_tables, &seq_lens})
    TORCH_CHECK_VALUE(t->is_contiguous(), "all inputs must be contiguous");
  const auto kd = key_cache.scalar_type();
  const bool fp8 = kd == at::kFloat8_e4m3fn;
  TORCH_CHECK_VALUE((kd == at::kHalf || kd == at::kBFloat16 || fp8) && value_cache.scalar_type() == kd,
                    "the caches must be FP16, BF16 or FP8-E4M3, both of one type");
  TORCH_CHECK_VALUE(fp8 == key_scales.has_value() && fp8 == value_scales.has_value(),
                    "key_scales and value_scales belong to an FP8-E4M3 cache, and to no other");
  TORCH_CHECK_VALUE(block_tables.scalar_type() == at::kInt && seq_lens.scalar_type() == at::kInt,
                    "block_tables and seq_lens must be int32");
  TORCH_CHECK_VALUE(key_cache.dim() == 4 && value_cache.sizes() == key_cache.sizes(),
                    "key_cache / value_cache must be 4-D and of one shape");
  const bool hnd = kv_layout == SQA_KV_HND;
  const int64_t hkv = key_cache.size(hnd ? 1 : 2);
  TORCH_CHECK_VALUE(key_cache.size(3) == kHeadDim, "the kernel supports head_dim 128");
  TORCH_CHECK_VALUE(key_cache.size(hnd ? 2 : 1) == kPage, "page_size must be 16");
  TORCH_CHECK_VALUE(block_tables.dim() == 2 && seq_lens.numel() == block_tables.size(0),
                    "invalid metadata: block_tables must be [batch, max_pages], seq_lens [batch]");
  TORCH_CHECK_VALUE(key_cache.size(0) > 0 && hkv > 0 && block_tables.size(1) > 0, "empty KV cache is not supported");
  TORCH_CHECK_VALUE(scores.scalar_type() == at::kFloat && scores.sizes() == at::IntArrayRef({key_cache.size(0), hkv, kPage}),
                    "scores must be a contiguous fp32 tensor [num_pages, Hkv, 16]");
  TORCH_CHECK_VALUE(budget >= 1 && budget <= (1 << 30), "budget must be in [1, 2^30]");
  TORCH_CHECK_VALUE(recent >= 0 && sinks >= 0 && recent <= budget && sinks <= budget - recent,
                    "recent and sinks must not be negative, and together at most budget");
  sqa_scales scales = {};
  if (fp8) scales = fill_scales(*key_scales, *value_scales, key_cache, hkv);
  const int64_t page_stride = cache_page_stride(key_cache, value_cache);
  const int64_t batch = block_tables.size(0);
  const at::Tensor lens = new_lens.has_value() ? *new_lens : at::empty_like(seq_lens);
  TORCH_CHECK_VALUE(lens.device() == dev && lens.scalar_type() == at::kInt && lens.is_contiguous() &&
                        lens.sizes() == seq_lens.sizes() && (batch == 0 || lens.data_ptr() != seq_lens.data_ptr()),
                    "new_lens must be a contiguous int32 tensor shaped like seq_lens, and another one");
  const at::Tensor from = kept.has_value() ? *kept : at::empty({batch, hkv, budget}, seq_lens.options());
  TORCH_CHECK_VALUE(from.device() == dev && from.scalar_type() == at::kInt && from.is_contiguous() &&
                        from.sizes() == at::IntArrayRef({batch, hkv, budget}),
                    "kept must be a contiguous int32 tensor [batch, Hkv, budget]");
  if (batch == 0) return {lens, from};
  c10::cuda::OptionalCUDAGuard guard;
  const cudaStream_t stream = on_device(guard, dev);
  const CallMemory mem = memory_for(kUseEvict, 256, dev, stream);
  const auto turn = mem.hold();
  const at::Tensor& word = mem.ws;
  sqa_evict_args a = {};
  a.key_cache = key_cache.data_ptr();
  a.value_cache = value_cache.data_ptr();
  a.scores = scores.data_ptr<float>();
  a.block_tables = block_tables.data_ptr<int32_t>();
  a.seq_lens = seq_lens.data_ptr<int32_t>();
  a.new_lens = lens.data_ptr<int32_t>();
  a.kept = from.data_ptr<int32_t>();
  a.status = static_cast<uint32_t*>(word.data_ptr());
  a.batch = (int32_t)batch;
  a.num_kv_heads = (int32_t)hkv;
  a.head_dim = (int32_t)kHeadDim;
  a.page_size = (int32_t)kPage;
  a.num_pages = (int32_t)key_cache.size(0);
  a.max_pages = (int32_t)block_tables.size(1);
  a.kv_layout = (int32_t)kv_layout;
  a.kv_dtype = fp8 ? SQA_KV_FP8_E4M3 : SQA_KV_SAME;
  a.budget = (int32_t)budget;
  a.recent = (int32_t)recent;
  a.sinks = (int32_t)sinks;
  a.page_stride = page_stride;
  if (check) clear_status(word, stream);
  check_status(sqa_cache_evict(&a, fp8 ? &scales : nullptr, stream), "sqa_cache_evict");
  if (check) raise_device_bits(word.data_ptr(), stream);
  return {lens, from};
}

// ---- the registered operators (functional: they allocate their outputs)
at::Tensor op_forward(const at::Tensor& query, const at::Tensor& key_cache, const at::Tensor& value_cache,
                      const at::Tensor& block_tables, const at::Tensor& seq_lens, int64_t page_size,
                      int64_t max_seq_len, int64_t kernel, int64_t kv_layout, double sm_scale, double out_scale) {
  return forward(query, key_cache, value_cache, block_tables, seq_lens, page_size, max_seq_len, c10::nullopt,
                 c10::nullopt, 0, 0, kernel, false, kv_layout, sm_scale, out_scale, 0, 0);
}

std::tuple<at::Tensor, at::Tensor> op_forward_partial(const at::Tensor& query, const at::Tensor& key_cache,
                                                      const at::Tensor& value_cache, const at::Tensor& block_tables,
                                                      const at::Tensor& seq_lens, int64_t page_size,
                                                      const c10::optional<at::Tensor>& mask_lens,
                                                      int64_t max_seq_len, int64_t kernel, int64_t kv_layout,
                                                      double sm_scale, double out_scale) {
  return forward_partial(query, key_cache, value_cache, block_tables, seq_lens, page_size, mask_lens, max_seq_len,
                         c10::nullopt, c10::nullopt, c10::nullopt, 0, 0, kernel, false, kv_layout, sm_scale,
                         out_scale, 0, 0);
}

std::tuple<at::Tensor, at::Tensor> op_forward_scaled(const at::Tensor& query, const at::Tensor& key_cache,
                                                     const at::Tensor& value_cache, const at::Tensor& key_scales,
                                                     const at::Tensor& value_scales, const at::Tensor& block_tables,
                                                     const at::Tensor& seq_lens, int64_t page_size, int64_t max_seq_len,
                                                     int64_t kv_layout, double sm_scale, double out_scale) {
  auto [o, l] = forward_scaled(query, key_cache, value_cache, key_scales, value_scales, block_tables, seq_lens, page_size,
                               c10::nullopt, max_seq_len, c10::nullopt, c10::nullopt, true, c10::nullopt, 0, false,
                               kv_layout, sm_scale, out_scale, 0, 0);
  return {o, *l};
}

std::tuple<at::Tensor, at::Tensor> meta_forward_scaled(const at::Tensor& query, const at::Tensor&, const at::Tensor&,
                                                       const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                                       const at::Tensor&, int64_t, int64_t, int64_t, double, double) {
  return {at::empty_like(query), at::empty(query.sizes().slice(0, 3), query.options().dtype(at::kFloat))};
}

at::Tensor meta_forward(const at::Tensor& query, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                        const at::Tensor&, int64_t, int64_t, int64_t, int64_t, double, double) {
  return at::empty_like(query);
}

std::tuple<at::Tensor, at::Tensor> meta_forward_partial(const at::Tensor& query, const at::Tensor&,
                                                        const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                                        int64_t, const c10::optional<at::Tensor>&, int64_t, int64_t,
                                                        int64_t, double, double) {
  const auto f32 = query.options().dtype(at::kFloat);
  return {at::empty(query.sizes(), f32), at::empty(query.sizes().slice(0, 3), f32)};
}

}  // namespace

TORCH_LIBRARY(sqa_b200, m) {
  m.def(
      "small_q_attention(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_tables, "
      "Tensor seq_lens, int page_size, int max_seq_len=0, int kernel=0, int kv_layout=0, float sm_scale=0., "
      "float out_scale=1.) -> Tensor");
  m.def(
      "small_q_attention_partial(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_tables, "
      "Tensor seq_lens, int page_size, Tensor? mask_lens=None, int max_seq_len=0, int kernel=0, int kv_layout=0, "
      "float sm_scale=0., float out_scale=1.) -> (Tensor, Tensor)");
  m.def(
      "small_q_attention_scaled(Tensor query, Tensor key_cache, Tensor value_cache, Tensor key_scales, "
      "Tensor value_scales, Tensor block_tables, Tensor seq_lens, int page_size, int max_seq_len=0, int kv_layout=0, "
      "float sm_scale=0., float out_scale=1.) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(sqa_b200, CUDA, m) {
  m.impl("small_q_attention", &op_forward);
  m.impl("small_q_attention_partial", &op_forward_partial);
  m.impl("small_q_attention_scaled", &op_forward_scaled);
}

TORCH_LIBRARY_IMPL(sqa_b200, Meta, m) {
  m.impl("small_q_attention", &meta_forward);
  m.impl("small_q_attention_partial", &meta_forward_partial);
  m.impl("small_q_attention_scaled", &meta_forward_scaled);
}

PYBIND11_MODULE(_sqa_torch, m) {
  m.doc() = "small-q paged MTP attention (B200): direct entry over the C ABI";
  m.def("forward", &forward, "causal paged MTP attention (see small_q_attention_b200.small_q_attention)");
  m.def("forward_partial", &forward_partial, "shard form: normalised fp32 O and natural-log LSE");
  m.def("forward_scaled", &forward_scaled, "attention over a block-scaled e4m3 cache", py::arg("query"),
        py::arg("key_cache"), py::arg("value_cache"), py::arg("key_scales"), py::arg("value_scales"),
        py::arg("block_tables"), py::arg("seq_lens"), py::arg("page_size"), py::arg("mask_lens"),
        py::arg("max_seq_len"), py::arg("out"), py::arg("out_lse"), py::arg("return_lse"), py::arg("workspace"),
        py::arg("num_ctas"), py::arg("check"), py::arg("kv_layout"), py::arg("sm_scale"), py::arg("out_scale"),
        py::arg("min_seq_len"), py::arg("cluster") = 0);
  m.def("append_scaled", &append_scaled, "quantising append to a block-scaled e4m3 cache");
  m.def("accumulate_weights", &accumulate_weights, "attention weight of every cached token, added to its score");
  m.def("cache_evict", &cache_evict, "keep the tokens of the highest scores within a budget, compacted in place");
  m.def("abi_version", &sqa_abi_version);
}
