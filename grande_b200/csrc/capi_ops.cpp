// extern "C" entry points of the operators on device memory (declared in
// include/omg_b200.h): argument checks, then the launches.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "capi_util.h"
#include "omg_b200.h"
#include "paged.cuh"
#include "sample.cuh"

using namespace omg;

namespace {

constexpr int kMaxDevices = 64;

// What the launches need to know of a device, looked up once.
struct DeviceInfo {
  int sms = 0;
};

const DeviceInfo& device_info(int device) {
  static std::mutex mu;
  static DeviceInfo info[kMaxDevices];
  std::lock_guard<std::mutex> g(mu);
  DeviceInfo& d = info[device];
  if (!d.sms) {
    int major = 0, minor = 0, sms = 0;
    CUDA_TRY(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device));
    CUDA_TRY(cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, device));
    if (major != 10 || minor != 0)
      fail("device %d is sm_%d%d; this library is built for sm_100a (B200)", device, major, minor);
    CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    DeviceScope on(device);
    paged_attention_setup_device();
    sample_setup_device();
    CUDA_TRY(cudaGetLastError());
    d.sms = sms;
  }
  return d;
}

void check_device(const char* op, int device) {
  if (device < 0 || device >= kMaxDevices) fail("%s: device %d", op, device);
}

void check_aligned(const char* op, const char* what, const void* p, size_t align) {
  if (!p) fail("%s: %s is null", op, what);
  if (reinterpret_cast<uintptr_t>(p) % align) fail("%s: %s is not %zu-byte aligned", op, what, align);
}

PagedCache to_cache(const char* op, const omg_paged_cache* c) {
  if (!c) fail("%s: cache is null", op);
  check_aligned(op, "cache rows", c->rows, 16);
  if (c->dtype != OMG_TYPE_F16 && c->dtype != OMG_TYPE_BF16)
    fail("%s: cache dtype %d (f16 or bf16)", op, c->dtype);
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256 && c->head_dim != 512)
    fail("%s: head_dim %d (64, 128, 256 or 512)", op, c->head_dim);
  if (c->kv_heads < 1 || c->kv_heads > 1024) fail("%s: kv_heads %d", op, c->kv_heads);
  int lg = 0;
  while ((1 << lg) < c->page_rows && lg < 9) ++lg;
  if (c->page_rows < 16 || c->page_rows > 256 || (1 << lg) != c->page_rows)
    fail("%s: page of %d rows (16, 32, 64, 128 or 256)", op, c->page_rows);
  // Row numbers are 32-bit in the kernels; bytes are 64-bit.
  if (c->n_pages < 1 || c->n_pages > ((int64_t(1) << 31) - 512) / c->page_rows)
    fail("%s: %lld pages of %d rows", op, static_cast<long long>(c->n_pages), c->page_rows);
  PagedCache o{};
  o.rows = c->rows;
  o.n_pages = c->n_pages;
  o.page_log2 = lg;
  o.kv_heads = c->kv_heads;
  o.hd = c->head_dim;
  o.dtype = c->dtype == OMG_TYPE_F16 ? kOpF16 : kOpBf16;
  return o;
}

PagedBatch to_batch(const char* op, const omg_paged_batch* b, const omg_paged_cache* c, int tokens,
                    bool prefix_pages) {
  if (!b) fail("%s: batch is null", op);
  if (b->n_seqs < 0 || b->n_groups < 0 || b->max_pages < 0 || b->max_prefix_pages < 0 || tokens < 0)
    fail("%s: negative batch size", op);
  const int64_t most = std::max(b->max_pages, b->max_prefix_pages);
  if (most * c->page_rows > (int64_t(1) << 30))
    fail("%s: %lld pages of %d rows per sequence", op, static_cast<long long>(most), c->page_rows);
  if (b->n_seqs > 0) {
    check_aligned(op, "q_start", b->q_start, 4);
    check_aligned(op, "lens", b->lens, 4);
    if (b->max_pages > 0) check_aligned(op, "pages", b->pages, 4);
  }
  if (b->n_groups > 0) {
    check_aligned(op, "group_start", b->group_start, 4);
    check_aligned(op, "prefix_lens", b->prefix_lens, 4);
    if (prefix_pages && b->max_prefix_pages > 0)
      check_aligned(op, "prefix_pages", b->prefix_pages, 4);
  }
  PagedBatch o{};
  o.q_start = b->q_start;
  o.lens = b->lens;
  o.pages = b->pages;
  o.group_start = b->group_start;
  o.prefix_lens = b->prefix_lens;
  o.prefix_pages = b->prefix_pages;
  o.n_seqs = b->n_seqs;
  o.n_groups = b->n_groups;
  o.max_pages = b->max_pages;
  o.max_prefix_pages = b->max_prefix_pages;
  o.tokens = tokens;
  return o;
}

// Shape of an attention call: everything but its pointers.
PagedAttnArgs attention_shape(const char* op, int device, const omg_paged_cache* cache,
                              const omg_paged_batch* batch, int tokens, int heads, size_t* bytes) {
  PagedAttnArgs a{};
  a.c = to_cache(op, cache);
  a.b = to_batch(op, batch, cache, tokens, true);
  if (heads < 1 || heads % a.c.kv_heads || heads / a.c.kv_heads > kPagedTileRows)
    fail("%s: %d query heads over %d KV heads", op, heads, a.c.kv_heads);
  a.heads = heads;
  if (!paged_attention_shape(&a))
    fail("%s: %d query rows of %d sequences in one call (split the batch)", op, tokens,
         batch->n_seqs);
  *bytes = paged_attention_layout(&a, device_info(device).sms);
  return a;
}

}  // namespace

extern "C" {

int omg_paged_append(int device, const omg_paged_cache* cache, const omg_paged_batch* batch,
                     const omg_append_args* p, void* stream) {
  return guarded([&]() -> int {
    const char* op = "omg_paged_append";
    check_device(op, device);
    if (!p) fail("%s: args is null", op);
    PagedAppendArgs a{};
    a.c = to_cache(op, cache);
    a.b = to_batch(op, batch, cache, p->tokens, false);
    if (p->heads < 1 || p->heads > 4096) fail("%s: heads %d", op, p->heads);
    const int hd = a.c.hd;
    const int64_t width = (int64_t(p->heads) + (p->has_kv ? 2 * a.c.kv_heads : 0)) * hd;
    if (p->qkv_dtype != OMG_TYPE_F32 && p->qkv_dtype != cache->dtype)
      fail("%s: qkv dtype %d (f32 or the cache's)", op, p->qkv_dtype);
    const int esz = p->qkv_dtype == OMG_TYPE_F32 ? 4 : 2;
    if (p->tokens > 0 && batch->n_seqs > 0) {
      check_aligned(op, "qkv", p->qkv, 16);
      check_aligned(op, "q_out", p->q_out, 16);
    }
    if (p->qkv_stride < width || p->qkv_stride * esz % 16)
      fail("%s: qkv stride %lld (at least %lld, rows 16-byte aligned)", op,
           static_cast<long long>(p->qkv_stride), static_cast<long long>(width));
    if (p->q_stride < int64_t(p->heads) * hd || p->q_stride * 2 % 16)
      fail("%s: q stride %lld (at least %lld, rows 16-byte aligned)", op,
           static_cast<long long>(p->q_stride), static_cast<long long>(p->heads) * hd);
    if (p->n_freq < 0 || p->n_freq > hd / 2)
      fail("%s: %d rotated pairs of head_dim %d", op, p->n_freq, hd);
    if (p->n_freq > 0) check_aligned(op, "inv_freq", p->inv_freq, 8);
    if (p->q_norm) check_aligned(op, "q_norm", p->q_norm, 16);
    if (p->k_norm) check_aligned(op, "k_norm", p->k_norm, 16);
    if (!(p->eps >= 0.f) || !std::isfinite(p->norm_offset) || !std::isfinite(p->q_scale))
      fail("%s: eps, norm_offset or q_scale", op);
    if (p->tokens == 0 || batch->n_seqs == 0) return 0;
    a.qkv = p->qkv;
    a.qkv_stride = p->qkv_stride;
    a.qkv_dtype = p->qkv_dtype == OMG_TYPE_F32 ? kOpF32 : a.c.dtype;
    a.heads = p->heads;
    a.has_kv = p->has_kv != 0;
    a.q_out = p->q_out;
    a.q_stride = p->q_stride;
    a.q_norm = p->q_norm;
    a.k_norm = p->k_norm;
    a.v_norm = p->v_norm != 0;
    a.norm_offset = p->norm_offset;
    a.eps = p->eps;
    a.q_scale = p->q_scale;
    a.inv_freq = p->inv_freq;
    a.n_freq = p->n_freq;
    DeviceScope on(device);
    launch_paged_append(a, device_info(device).sms, static_cast<cudaStream_t>(stream));
    CUDA_TRY(cudaGetLastError());
    return 0;
  });
}

size_t omg_paged_attention_workspace(int device, const omg_paged_cache* cache,
                                     const omg_paged_batch* batch, int tokens, int heads) {
  size_t bytes = 0;
  const int rc = guarded([&]() -> int {
    const char* op = "omg_paged_attention_workspace";
    check_device(op, device);
    attention_shape(op, device, cache, batch, tokens, heads, &bytes);
    return 0;
  });
  return rc == 0 ? bytes : 0;
}

int omg_paged_attention(int device, const omg_paged_cache* cache, const omg_paged_batch* batch,
                        const omg_attention_args* p, void* workspace, size_t workspace_bytes,
                        void* stream) {
  return guarded([&]() -> int {
    const char* op = "omg_paged_attention";
    check_device(op, device);
    if (!p) fail("%s: args is null", op);
    if (!(p->scale > 0.f) || !std::isfinite(p->scale)) fail("%s: scale %g", op, p->scale);
    if (p->window < 0 || p->window > (1 << 30)) fail("%s: window %d", op, p->window);
    size_t need = 0;
    PagedAttnArgs a = attention_shape(op, device, cache, batch, p->tokens, p->heads, &need);
    const int64_t width = int64_t(p->heads) * a.c.hd;
    if (p->q_stride < width || p->q_stride % 8 || p->out_stride < width || p->out_stride % 8)
      fail("%s: q stride %lld, out stride %lld (at least %lld, rows 16-byte aligned)", op,
           static_cast<long long>(p->q_stride), static_cast<long long>(p->out_stride),
           static_cast<long long>(width));
    if (p->tokens == 0 || batch->n_seqs == 0) return 0;
    check_aligned(op, "q", p->q, 16);
    check_aligned(op, "out", p->out, 16);
    // (At head_dim 512 two CTAs read a row's q, and one may be done first.)
    if (p->q == p->out) fail("%s: out is q", op);
    check_aligned(op, "workspace", workspace, 256);
    if (workspace_bytes < need)
      fail("%s: workspace of %zu bytes, %zu needed", op, workspace_bytes, need);
    a.out = p->out;
    a.out_stride = p->out_stride;
    a.window = p->window;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    paged_attention_workspace(&a, workspace);
    DeviceScope on(device);
    PagedMaps maps;
    char err[256];
    if (!paged_attention_maps(a, p->q, p->q_stride, &maps, err, sizeof err))
      fail("%s: %s", op, err);
    launch_paged_attention(a, maps, static_cast<cudaStream_t>(stream));
    CUDA_TRY(cudaGetLastError());
    return 0;
  });
}

int omg_sample(int device, const omg_sample_args* p, void* stream) {
  return guarded([&]() -> int {
    const char* op = "omg_sample";
    check_device(op, device);
    if (!p) fail("%s: args is null", op);
    if (p->dtype != OMG_TYPE_F32 && p->dtype != OMG_TYPE_F16 && p->dtype != OMG_TYPE_BF16)
      fail("%s: dtype %d", op, p->dtype);
    SampleArgs a{};
    a.dtype = p->dtype == OMG_TYPE_F32 ? kOpF32 : p->dtype == OMG_TYPE_F16 ? kOpF16 : kOpBf16;
    if (p->rows < 0 || p->rows > (1 << 24)) fail("%s: %d rows", op, p->rows);
    if (p->vocab < 1 || p->vocab > sample_max_vocab())
      fail("%s: vocabulary of %d (1 to %d)", op, p->vocab, sample_max_vocab());
    if (p->stride < p->vocab)
      fail("%s: stride %lld < vocabulary %d", op, static_cast<long long>(p->stride), p->vocab);
    if (p->rows == 0) return 0;
    check_aligned(op, "logits", p->logits, p->dtype == OMG_TYPE_F32 ? 4 : 2);
    check_aligned(op, "u", p->u, 4);
    check_aligned(op, "tokens", p->tokens, 4);
    a.logits = p->logits;
    a.stride = p->stride;
    a.rows = p->rows;
    a.vocab = p->vocab;
    a.u = p->u;
    a.temperature = p->temperature;
    a.top_k = p->top_k;
    a.top_p = p->top_p;
    a.min_p = p->min_p;
    a.temperature1 = p->temperature_all;
    a.top_k1 = p->top_k_all;
    a.top_p1 = p->top_p_all;
    a.min_p1 = p->min_p_all;
    a.tokens = p->tokens;
    a.probs = p->probs;
    DeviceScope on(device);
    launch_sample(a, device_info(device).sms, static_cast<cudaStream_t>(stream));
    CUDA_TRY(cudaGetLastError());
    return 0;
  });
}

}  // extern "C"
