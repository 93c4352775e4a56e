// PyTorch side of the paged cache: argument checks, outputs, workspace, the current stream.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/types.h>

#include "paged.h"

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

namespace {

// Arguments that are wrong by themselves: the Python side turns this error into a ValueError. (What the kernels
// cannot take, a device, strides or a type, stays a RuntimeError.)
#define ME_CHECK_VALUE(cond, ...) TORCH_CHECK(cond, "value: ", __VA_ARGS__)

std::string shape(const Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}
std::string text(int64_t v) { return std::to_string(v); }

bool aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

me::PagedCache check_cache(const Tensor& k, const Tensor& v) {
  TORCH_CHECK(k.is_cuda() && v.is_cuda() && k.device() == v.device(), "k_pages and v_pages: CUDA tensors on one device are needed");
  TORCH_CHECK(k.scalar_type() == torch::kBFloat16 && v.scalar_type() == torch::kBFloat16, "k_pages and v_pages: bfloat16 is needed, got ",
              k.scalar_type(), " and ", v.scalar_type());
  ME_CHECK_VALUE(k.dim() == 4 && k.sizes() == v.sizes() && k.numel() > 0, "k_pages and v_pages: [pages, heads, page, dim] each is needed, got ",
                 shape(k), " and ", shape(v));
  const int64_t pages = k.size(0), heads = k.size(1), page = k.size(2), dim = k.size(3);
  ME_CHECK_VALUE(page == 16 || page == 32 || page == 64 || page == 128, "k_pages: pages of 16, 32, 64 or 128 positions are needed, got ", text(page));
  ME_CHECK_VALUE(dim == 64 || dim == 128 || dim == 256 || dim == 512, "k_pages: a head dimension of 64, 128, 256 or 512 is needed, got ", text(dim));
  ME_CHECK_VALUE(heads <= 4096 && pages < (1ll << 31), "k_pages: at most 4096 heads and 2^31 - 1 pages, got ", shape(k));
  for (const Tensor* t : {&k, &v}) {
    TORCH_CHECK(t->stride(3) == 1 && t->stride(2) == dim && (heads == 1 || t->stride(1) == page * dim) &&
                    (pages == 1 || (t->stride(0) >= heads * page * dim && t->stride(0) % 8 == 0)) && aligned(*t),
                "k_pages and v_pages: the elements of a page have to be contiguous, pages a multiple of 8 elements apart, 16-byte aligned");
  }
  const int64_t whole = heads * page * dim;
  return {k.data_ptr(), v.data_ptr(), pages == 1 ? whole : k.stride(0), pages == 1 ? whole : v.stride(0), (int)pages, (int)heads, (int)page, (int)dim};
}

// Whether a page of keys lies over one of values. Pages of each are in order of their addresses.
bool overlap(const me::PagedCache& c) {
  const int64_t whole = (int64_t)c.heads * c.page * c.dim;  // elements
  const int64_t k = reinterpret_cast<intptr_t>(c.k) / 2, v = reinterpret_cast<intptr_t>(c.v) / 2;
  if (k + (c.pages - 1) * c.k_stride + whole <= v || v + (c.pages - 1) * c.v_stride + whole <= k) return false;
  if (c.k_stride == c.v_stride) {  // each other's gaps
    const int64_t by = ((v - k) % c.k_stride + c.k_stride) % c.k_stride;
    return by < whole || by > c.k_stride - whole;
  }
  for (int64_t i = 0, j = 0; i < c.pages && j < c.pages;) {
    const int64_t by = v + j * c.v_stride - (k + i * c.k_stride);
    if (by > -whole && by < whole) return true;
    by > 0 ? ++i : ++j;
  }
  return false;
}

// int32: a number outside its range is no page and no position, and must not come back as another one.
Tensor narrow(const Tensor& t) { return t.scalar_type() == torch::kInt ? t : t.clamp(-1, INT32_MAX).to(torch::kInt); }

Tensor check_int(const Tensor& t, const Tensor& like, const char* what) {
  TORCH_CHECK(t.device() == like.device(), what, ": on another device than the pages");
  ME_CHECK_VALUE(t.scalar_type() == torch::kInt || t.scalar_type() == torch::kLong, what, ": int32 or int64 is needed, got ", t.scalar_type());
  return narrow(t).contiguous();
}

struct Batch {
  Tensor cu, lens, table;
  me::PagedBatch args;
};

Batch check_batch(const Tensor& pages, const Tensor& table, const Tensor& cu, const Tensor& lens, int64_t tokens) {
  ME_CHECK_VALUE(lens.dim() == 1 && cu.dim() == 1 && cu.size(0) == lens.size(0) + 1, "cu_seqlens, seq_lens: [sequences + 1] and [sequences] are needed, got ",
                 shape(cu), " and ", shape(lens));
  ME_CHECK_VALUE(table.dim() == 2 && table.size(0) == lens.size(0), "block_table: [sequences, pages of the longest] is needed, got ", shape(table),
                 " for ", text(lens.size(0)), " sequences");
  ME_CHECK_VALUE(table.size(1) * pages.size(2) <= INT32_MAX - (1 << 20), "block_table: rows of at most 2^31 - 2^20 positions, got ", text(table.size(1)), " pages");
  ME_CHECK_VALUE(tokens < (1 << 24) && lens.size(0) < (1 << 24), "at most 2^24 - 1 new tokens and sequences, got ", text(tokens));
  Batch b;
  b.cu = check_int(cu, pages, "cu_seqlens");
  b.lens = check_int(lens, pages, "seq_lens");
  TORCH_CHECK(table.device() == pages.device(), "block_table: on another device than the pages");
  ME_CHECK_VALUE(table.scalar_type() == torch::kInt || table.scalar_type() == torch::kLong, "block_table: int32 or int64 is needed, got ", table.scalar_type());
  b.table = table.scalar_type() == torch::kInt && (table.size(1) <= 1 || table.stride(1) == 1) ? table : narrow(table).contiguous();
  b.args = {b.cu.data_ptr<int>(), b.lens.data_ptr<int>(), b.table.data_ptr<int>(), b.table.stride(0), (int)table.size(1), (int)lens.size(0), (int)tokens};
  return b;
}

const float* check_weight(const Tensor& w, const Tensor& pages, int64_t n, const char* what) {
  TORCH_CHECK(w.device() == pages.device() && w.scalar_type() == torch::kFloat32 && w.is_contiguous(), what,
              ": contiguous float32 on the pages' device is needed");
  ME_CHECK_VALUE(w.dim() == 1 && w.size(0) == n, what, ": [", text(n), "] is needed, got ", shape(w));
  return w.data_ptr<float>();
}

int sms() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

// Heads [T, H, D] as the kernels and their tensor maps take them: contiguous, a multiple of 8 elements apart.
bool rows_fit(const Tensor& t) {
  auto fits = [&](int i) { return t.size(i) <= 1 || (t.stride(i) > 0 && t.stride(i) % 8 == 0); };
  return t.stride(2) == 1 && fits(0) && fits(1) && aligned(t);
}
// ... and as they are written: no two of them share memory.
bool apart(const Tensor& t) {
  const int64_t n = t.size(0), h = t.size(1), d = t.size(2);
  if (n <= 1 || h <= 1) return (n <= 1 || t.stride(0) >= d) && (h <= 1 || t.stride(1) >= d);
  return t.stride(1) <= t.stride(0) ? t.stride(1) >= d && t.stride(0) >= (h - 1) * t.stride(1) + d
                                    : t.stride(0) >= d && t.stride(1) >= (n - 1) * t.stride(0) + d;
}
int64_t head_stride(const Tensor& t) { return t.size(1) <= 1 ? t.size(2) : t.stride(1); }
int64_t token_stride(const Tensor& t) { return t.size(0) <= 1 ? t.size(1) * t.size(2) : t.stride(0); }

}  // namespace

Tensor paged_append(Tensor qkv, Tensor q_w, Tensor k_w, Tensor inv_freq, Tensor k_pages, Tensor v_pages, Tensor table, Tensor cu, Tensor lens,
                    int64_t q_heads, bool kv_shared, double eps) {
  me::AppendArgs a;
  a.cache = check_cache(k_pages, v_pages);
  const int64_t dim = a.cache.dim, heads = a.cache.heads;
  const c10::cuda::CUDAGuard guard(k_pages.device());
  TORCH_CHECK(qkv.device() == k_pages.device() && qkv.scalar_type() == torch::kBFloat16, "qkv: bfloat16 on the pages' device is needed");
  ME_CHECK_VALUE(q_heads >= 1 && q_heads <= 65536, "q_heads: 1 to 65536, got ", text(q_heads));
  ME_CHECK_VALUE(qkv.dim() == 2 && qkv.size(1) == (q_heads + (kv_shared ? 1 : 2) * heads) * dim, "qkv: [tokens, (q heads + ", kv_shared ? "" : "2 ",
                 "kv heads) dim] = [tokens, ", text((q_heads + (kv_shared ? 1 : 2) * heads) * dim), "] is needed, got ", shape(qkv));
  const int64_t tokens = qkv.size(0);
  const Batch batch = check_batch(k_pages, table, cu, lens, tokens);
  a.batch = batch.args;
  a.q_w = check_weight(q_w, k_pages, dim, "q_w");
  a.k_w = check_weight(k_w, k_pages, dim, "k_w");
  a.inv_freq = check_weight(inv_freq, k_pages, dim / 2, "inv_freq");
  if (!(qkv.stride(1) == 1 && (tokens <= 1 || qkv.stride(0) % 8 == 0) && aligned(qkv))) qkv = qkv.clone(at::MemoryFormat::Contiguous);
  a.qkv = qkv.data_ptr();
  a.qkv_stride = qkv.stride(0);
  Tensor q = torch::empty({tokens, q_heads, dim}, qkv.options().requires_grad(false));
  a.q = q.data_ptr();
  a.q_heads = (int)q_heads;
  a.kv_shared = kv_shared;
  a.eps = (float)eps;
  ME_CHECK_VALUE(!overlap(a.cache), "k_pages and v_pages: they lie over one another, and both are written");
  if (tokens == 0) return q;
  // the kernel writes through the pointers: a graph that has saved the pages learns of it by their versions
  k_pages.unsafeGetTensorImpl()->bump_version();
  v_pages.unsafeGetTensorImpl()->bump_version();
  me::launch_paged_append(a, sms(), at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return q;
}

std::vector<Tensor> paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor table, Tensor cu, Tensor lens, int64_t window, double scale,
                                    int64_t max_q, OptTensor out) {
  me::PagedAttentionArgs a;
  a.cache = check_cache(k_pages, v_pages);
  const int64_t dim = a.cache.dim, heads = a.cache.heads;
  const c10::cuda::CUDAGuard guard(k_pages.device());
  TORCH_CHECK(q.device() == k_pages.device() && q.scalar_type() == torch::kBFloat16, "q: bfloat16 on the pages' device is needed");
  ME_CHECK_VALUE(q.dim() == 3 && q.size(2) == dim, "q: [tokens, heads, ", text(dim), "] is needed, got ", shape(q));
  const int64_t tokens = q.size(0), q_heads = q.size(1);
  ME_CHECK_VALUE(q_heads >= heads && q_heads % heads == 0 && q_heads / heads <= 128, "q: heads a multiple of the pages' ", text(heads),
                 " (up to 128 times) are needed, got ", text(q_heads));
  ME_CHECK_VALUE(tokens * q_heads < (1ll << 31), "q: fewer than 2^31 rows (tokens times heads) are needed, got ", shape(q));
  ME_CHECK_VALUE(window >= 0 && window <= INT32_MAX, "window: a positive number or None, got ", text(window));
  // (the kernels take scores by powers of 2: scale / ln 2 has to be a number in 32 bits)
  ME_CHECK_VALUE((float)scale > 0 && (float)scale < 0x1p127f, "scale: a positive number (in 32 bits) below 2^127 is needed");
  ME_CHECK_VALUE(max_q >= 0, "max_q: a positive number or None, got ", text(max_q));
  const Batch batch = check_batch(k_pages, table, cu, lens, tokens);
  a.batch = batch.args;
  const Tensor given = q;
  if (!rows_fit(q)) q = q.clone(at::MemoryFormat::Contiguous);
  Tensor o;
  if (out.has_value()) {
    o = *out;
    // (units read rows of q that others' rows of o may lie over by then; q itself, not its copy above)
    ME_CHECK_VALUE(!o.numel() || !o.is_alias_of(given), "out: a tensor of its own is needed, not q's memory");
    ME_CHECK_VALUE(o.sizes() == q.sizes(), "out: q's shape ", shape(q), " is needed, got ", shape(o));
    TORCH_CHECK(o.device() == q.device() && o.scalar_type() == torch::kBFloat16 && rows_fit(o) && apart(o) && !o.is_alias_of(k_pages) && !o.is_alias_of(v_pages),
                "out: bfloat16 on the pages' device is needed, heads contiguous, a multiple of 8 elements and at least dim apart, 16-byte aligned, "
                "not the pages");
    o.unsafeGetTensorImpl()->bump_version();
  } else {
    o = torch::empty({tokens, q_heads, dim}, q.options().requires_grad(false));
  }
  Tensor lse = torch::empty({q_heads, tokens}, q.options().dtype(torch::kFloat32).requires_grad(false));
  if (tokens == 0) return {o, lse};
  a.q = q.data_ptr();
  a.q_token = token_stride(q), a.q_head = head_stride(q);
  a.o = o.data_ptr();
  a.o_token = token_stride(o), a.o_head = head_stride(o);
  a.lse = lse.data_ptr<float>();
  a.q_heads = (int)q_heads;
  a.window = (int)window;
  a.scale = (float)scale;
  a.clear_rest = !out.has_value();
  a.max_q = (int)std::min(max_q ? max_q : tokens, tokens);
  Tensor workspace = torch::empty({me::paged_attention_workspace(a, sms())}, q.options().dtype(torch::kByte).requires_grad(false));
  const char* wrong = me::launch_paged_attention(a, workspace.data_ptr(), sms(), at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(wrong == nullptr, "paged_attention: ", wrong);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {o, lse};
}

// (blocks, where): blocks of the attention kernels on this device in which a wait ran out since the process began, and where the last of them
// waited; what the device's current stream has ahead is in it.
std::vector<int64_t> paged_status(int64_t device) {
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  TORCH_CHECK(at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None,
              "paged_status: it waits for the current stream, which is being captured");
  int words[2] = {0, 0};
  C10_CUDA_CHECK(me::paged_waits(words, at::cuda::getCurrentCUDAStream()));
  return {words[0], words[1]};
}
