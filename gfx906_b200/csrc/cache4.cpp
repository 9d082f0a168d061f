// Torch operators of the paged 4-bit key/value cache over its C ABI
// (include/gfx906_b200_cache4.h). Like `attn`: inputs are checked, launched on
// the current stream of their device, and failures raise RuntimeError.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/gfx906_b200_cache4.h"

using torch::Tensor;

namespace {

constexpr int64_t kPage = 64;

void check_int32(const Tensor& t, const Tensor& on, int64_t dim, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == on.device() && t.dtype() == torch::kInt32 && t.dim() == dim &&
                  t.is_contiguous(),
              "cache4: ", name, " must be a contiguous ", std::to_string(dim), "-dimensional int32 CUDA tensor on the other tensors' device");
}

// [pages, kv_heads, 72 D] uint8 -> (pages, kv_heads, D)
std::tuple<int, int, int> check_cache(const Tensor& cache) {
  TORCH_CHECK(cache.is_cuda() && cache.dtype() == torch::kUInt8 && cache.dim() == 3 && cache.is_contiguous(),
              "cache4: cache must be a contiguous uint8 CUDA tensor [pages, kv_heads, page_bytes]");
  const int64_t D = cache.size(2) / 72;
  TORCH_CHECK((D == 64 || D == 128) && cache.size(2) == 72 * D,
              "cache4: cache pages must have 72 * head_dim bytes, head_dim 64 or 128");
  TORCH_CHECK(cache.size(0) <= INT32_MAX / kPage && cache.size(1) >= 1 && cache.size(1) <= INT32_MAX,
              "cache4: cache is too large or has no heads");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(cache.data_ptr()) % 16 == 0, "cache4: cache must start on 16 bytes");
  return {static_cast<int>(cache.size(0)), static_cast<int>(cache.size(1)), static_cast<int>(D)};
}

const float* check_scale(const std::optional<Tensor>& s, const Tensor& on, int64_t heads, const char* name) {
  if (!s.has_value()) return nullptr;
  TORCH_CHECK(s->is_cuda() && s->device() == on.device() && s->dtype() == torch::kFloat32 && s->is_contiguous() &&
                  s->dim() == 1 && s->size(0) == heads,
              "cache4: ", name, " must be a contiguous float32 CUDA tensor [kv_heads] on the cache's device");
  return s->data_ptr<float>();
}

int dtype_code(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && (t.dtype() == torch::kHalf || t.dtype() == torch::kBFloat16),
              "cache4: ", name, " must be a float16 or bfloat16 CUDA tensor");
  return t.dtype() == torch::kBFloat16 ? 1 : 0;
}

// Elements from one token (dim 0) or head (dim 1) to the next. A dimension of one
// entry may have any stride in torch; no kernel uses it.
int64_t stride_of(const Tensor& t, int dim) { return t.size(dim) == 1 ? t.size(2) : t.stride(dim); }

// Rows the kernels can load 16 bytes at a time: contiguous in the head dim,
// starting on 16 bytes. Anything else is copied once.
bool rows_ok(const Tensor& t) {
  return t.stride(2) == 1 && stride_of(t, 0) % 8 == 0 && stride_of(t, 1) % 8 == 0 &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}
Tensor with_rows(const Tensor& t) {
  if (t.numel() == 0 || rows_ok(t)) return t;
  // a contiguous view may start off 16 bytes
  return t.is_contiguous() ? t.clone(at::MemoryFormat::Contiguous) : t.contiguous();
}

// Where the rows [tokens, heads] of a tensor start, in elements.
struct RowGrid {
  int64_t at, step_t, step_h;
  explicit RowGrid(const Tensor& t)
      : at(reinterpret_cast<intptr_t>(t.data_ptr()) / 2), step_t(stride_of(t, 0)), step_h(stride_of(t, 1)) {}
};
// Do two different rows of D elements of one grid share an element? Of two rows
// dh >= 0 heads apart the nearest are those whose distance in tokens makes up for it.
bool rows_meet(const RowGrid& a, int64_t T, int64_t H, int64_t D, int64_t offset, bool same) {
  for (int64_t dh = same ? 0 : 1 - H; dh < H; ++dh) {
    const int64_t far = offset + dh * a.step_h;
    if (same && dh == 0) {
      if (T > 1 && a.step_t < D) return true;
      continue;
    }
    const int64_t near = a.step_t ? -far / a.step_t : 0;
    for (int64_t dt = near - 1; dt <= near + 1; ++dt)
      if (std::abs(dt) < T && std::abs(far + dt * a.step_t) < D) return true;
  }
  return false;
}
// Rows of out that are not its own, or that are rows of q other than the same ones:
// calls write rows while others are still read.
bool out_ok(const Tensor& out, const Tensor& q) {
  const int64_t T = q.size(0), H = q.size(1), D = q.size(2);
  if (q.numel() == 0) return true;
  const RowGrid o(out), x(q);
  if (!(o.step_h >= D && o.step_t >= (H - 1) * o.step_h + D) && rows_meet(o, T, H, D, 0, true)) return false;
  const auto end = [&](const RowGrid& g) { return g.at + (T - 1) * g.step_t + (H - 1) * g.step_h + D; };
  if (o.at >= end(x) || x.at >= end(o)) return true;
  if (o.step_t == x.step_t && o.step_h == x.step_h) return o.at == x.at || !rows_meet(o, T, H, D, o.at - x.at, false);
  // two orders in one piece of memory: every row of one against its neighbours in the other
  std::vector<int64_t> rows;
  rows.reserve(T * H);
  for (int64_t t = 0; t < T; ++t)
    for (int64_t h = 0; h < H; ++h) rows.push_back(x.at + t * x.step_t + h * x.step_h);
  std::sort(rows.begin(), rows.end());
  for (int64_t t = 0; t < T; ++t)
    for (int64_t h = 0; h < H; ++h) {
      const int64_t row = o.at + t * o.step_t + h * o.step_h;
      const auto next = std::upper_bound(rows.begin(), rows.end(), row - D);
      if (next != rows.end() && *next < row + D) return false;
    }
  return true;
}

// These calls are as short as their launches, so results are allocated without
// the dispatcher, and the index tensors of a plan at once.
Tensor new_tensor(c10::IntArrayRef sizes, c10::ScalarType type, const Tensor& on) {
  return at::detail::empty_cuda(sizes, type, on.device(), std::nullopt);
}
// A contiguous tensor in `all`, from element `at` on.
Tensor part_of(const Tensor& all, int64_t at, c10::IntArrayRef sizes) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(all.storage()), all.key_set(),
                                                      all.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(at);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

// Scratch memory of one call, from the caching allocator: calls on other streams
// and other captured graphs never share it.
class Workspace {
 public:
  Workspace(size_t bytes, cudaStream_t stream)
      : p_(bytes ? c10::cuda::CUDACachingAllocator::raw_alloc_with_stream(bytes, stream) : nullptr) {}
  ~Workspace() {
    if (p_) c10::cuda::CUDACachingAllocator::raw_delete(p_);
  }
  Workspace(const Workspace&) = delete;
  void* get() const { return p_; }

 private:
  void* p_;
};

void check_status(int rc) { TORCH_CHECK(rc == GFX906_B200_OK, "cache4: ", gfx906_b200_attn_error_string(rc)); }

}  // namespace

using PlanOut = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

PlanOut cache4_plan(Tensor tables, Tensor lengths, Tensor counts, Tensor free_pages, Tensor free_count, int64_t tokens) {
  check_int32(tables, tables, 2, "tables");
  check_int32(lengths, tables, 1, "lengths");
  check_int32(counts, tables, 1, "counts");
  check_int32(free_pages, tables, 1, "free_pages");
  check_int32(free_count, tables, 1, "free_count");
  const int64_t R = tables.size(0), W = tables.size(1);
  TORCH_CHECK(lengths.size(0) == R && counts.size(0) == R && free_count.size(0) == 1,
              "cache4: lengths and counts must have one entry per row of tables, free_count one entry");
  TORCH_CHECK(R <= 8192, "cache4: at most 8192 requests");
  TORCH_CHECK(W <= INT32_MAX / kPage && R * W <= INT32_MAX && free_pages.size(0) <= INT32_MAX, "cache4: sizes are too large");
  TORCH_CHECK(tokens >= 0 && tokens < INT32_MAX, "cache4: tokens must be a non-negative int32");
  const c10::cuda::CUDAGuard guard(tables.device());
  const Tensor all = new_tensor({3 * R + 2 * tokens + 2}, torch::kInt32, tables);
  int64_t at = 0;
  auto cut = [&](int64_t n) {
    at += n;
    return part_of(all, at - n, {n});
  };
  Tensor query_start = cut(R + 1), lengths_out = cut(R), added = cut(R), slots = cut(tokens), positions = cut(tokens),
         free_out = cut(1);
  check_status(gfx906_b200_cache4_plan(
      tables.data_ptr<int>(), lengths.data_ptr<int>(), counts.data_ptr<int>(), free_pages.data_ptr<int>(),
      free_count.data_ptr<int>(), static_cast<int>(R), static_cast<int>(W), static_cast<int>(free_pages.size(0)),
      static_cast<int>(tokens), query_start.data_ptr<int>(), lengths_out.data_ptr<int>(), added.data_ptr<int>(),
      slots.data_ptr<int>(), positions.data_ptr<int>(), free_out.data_ptr<int>(), at::cuda::getCurrentCUDAStream()));
  return {query_start, lengths_out, added, slots, positions, free_out};
}

void cache4_write(Tensor k, Tensor v, Tensor cache, Tensor slots, std::optional<Tensor> k_scale,
                  std::optional<Tensor> v_scale) {
  const auto [pages, heads, D] = check_cache(cache);
  const int dtype = dtype_code(k, "k");
  TORCH_CHECK(v.is_cuda() && v.dtype() == k.dtype(), "cache4: k and v must have the same dtype");
  TORCH_CHECK(k.device() == cache.device() && v.device() == cache.device(), "cache4: k, v and cache must be on the same device");
  TORCH_CHECK(k.dim() == 3 && v.sizes() == k.sizes() && k.size(1) == heads && k.size(2) == D,
              "cache4: k and v must be [tokens, kv_heads, head_dim] like the cache");
  check_int32(slots, cache, 1, "slots");
  TORCH_CHECK(slots.size(0) == k.size(0) && k.size(0) <= INT32_MAX, "cache4: one slot per token");
  const float* ks = check_scale(k_scale, cache, heads, "k_scale");
  const float* vs = check_scale(v_scale, cache, heads, "v_scale");
  const c10::cuda::CUDAGuard guard(cache.device());
  const Tensor kc = with_rows(k), vc = with_rows(v);
  check_status(gfx906_b200_cache4_write(kc.data_ptr(), vc.data_ptr(), dtype, stride_of(kc, 0), stride_of(kc, 1),
                                        stride_of(vc, 0), stride_of(vc, 1), static_cast<int>(k.size(0)), heads, D,
                                        cache.data_ptr(), pages, slots.data_ptr<int>(), ks, vs,
                                        at::cuda::getCurrentCUDAStream()));
}

std::tuple<Tensor, Tensor> cache4_read(Tensor cache, Tensor slots, std::optional<Tensor> k_scale,
                                       std::optional<Tensor> v_scale, int64_t dtype) {
  const auto [pages, heads, D] = check_cache(cache);
  check_int32(slots, cache, 1, "slots");
  TORCH_CHECK(slots.size(0) <= INT32_MAX && dtype >= 0 && dtype <= 2, "cache4: too many slots or unknown dtype");
  const float* ks = check_scale(k_scale, cache, heads, "k_scale");
  const float* vs = check_scale(v_scale, cache, heads, "v_scale");
  const c10::cuda::CUDAGuard guard(cache.device());
  const auto type = dtype == 0 ? torch::kHalf : dtype == 1 ? torch::kBFloat16 : torch::kFloat32;
  Tensor k = new_tensor({slots.size(0), heads, D}, type, cache), v = new_tensor({slots.size(0), heads, D}, type, cache);
  check_status(gfx906_b200_cache4_read(cache.data_ptr(), pages, slots.data_ptr<int>(), ks, vs,
                                       static_cast<int>(slots.size(0)), heads, D, k.data_ptr(), v.data_ptr(),
                                       static_cast<int>(dtype), at::cuda::getCurrentCUDAStream()));
  return {k, v};
}

Tensor attn_cache4(Tensor q, Tensor cache, Tensor tables, Tensor lengths, Tensor query_start, double scale, bool causal,
                   std::optional<Tensor> k_scale, std::optional<Tensor> v_scale, std::optional<int64_t> max_tokens,
                   std::optional<Tensor> out) {
  const auto [pages, kv_heads, D] = check_cache(cache);
  const int dtype = dtype_code(q, "q");
  TORCH_CHECK(q.device() == cache.device(), "cache4: q and cache must be on the same device");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == D && q.size(1) >= 1 && q.size(1) % kv_heads == 0 && q.size(0) <= INT32_MAX &&
                  q.size(0) * (q.size(1) / kv_heads) <= INT32_MAX,
              "cache4: q must be [tokens, heads, head_dim], heads a multiple of the cache's");
  check_int32(tables, cache, 2, "tables");
  check_int32(lengths, cache, 1, "lengths");
  check_int32(query_start, cache, 1, "query_start");
  const int64_t R = tables.size(0), W = tables.size(1);
  TORCH_CHECK(lengths.size(0) == R && query_start.size(0) == R + 1,
              "cache4: lengths must have one entry per row of tables, query_start one more");
  TORCH_CHECK(R <= 8192 && W <= INT32_MAX / kPage, "cache4: at most 8192 requests; tables too wide");
  TORCH_CHECK(std::isfinite(scale) && std::isfinite(static_cast<float>(scale)), "cache4: scale must be finite");
  TORCH_CHECK(!max_tokens.has_value() || *max_tokens >= 0, "cache4: max_tokens must not be negative");
  const float* ks = check_scale(k_scale, cache, kv_heads, "k_scale");
  const float* vs = check_scale(v_scale, cache, kv_heads, "v_scale");
  if (out.has_value()) {
    TORCH_CHECK(out->is_cuda() && out->device() == q.device() && out->dtype() == q.dtype() && out->sizes() == q.sizes() &&
                    rows_ok(*out),
                "cache4: out must be a tensor like q with rows that start on 16 bytes");
  }
  const c10::cuda::CUDAGuard guard(cache.device());
  const Tensor qc = with_rows(q);
  TORCH_CHECK(!out.has_value() || out_ok(*out, qc), "cache4: out must have rows of its own: q itself, or no row of q");
  Tensor o = out.has_value() ? *out : new_tensor(q.sizes(), q.scalar_type(), q);
  if (q.numel() == 0) return o;
  gfx906_b200_cache4_attn_args g{};
  g.q = qc.data_ptr();
  g.o = o.data_ptr();
  g.cache = cache.data_ptr();
  g.tables = tables.data_ptr<int>();
  g.lengths = lengths.data_ptr<int>();
  g.query_start = query_start.data_ptr<int>();
  g.k_scale = ks;
  g.v_scale = vs;
  g.q_stride_t = stride_of(qc, 0);
  g.q_stride_h = stride_of(qc, 1);
  g.o_stride_t = stride_of(o, 0);
  g.o_stride_h = stride_of(o, 1);
  g.dtype = dtype;
  g.tokens = static_cast<int>(q.size(0));
  g.heads = static_cast<int>(q.size(1));
  g.kv_heads = kv_heads;
  g.D = D;
  g.pages = pages;
  g.requests = static_cast<int>(R);
  g.width = static_cast<int>(W);
  g.max_tokens = static_cast<int>(std::min<int64_t>(max_tokens.value_or(q.size(0)), q.size(0)));
  g.causal = causal ? 1 : 0;
  g.zero_rest = out.has_value() ? 0 : 1;
  g.scale = static_cast<float>(scale);
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const size_t bytes = gfx906_b200_cache4_attn_workspace_size(&g);
  const Workspace ws(bytes, stream);
  check_status(gfx906_b200_cache4_attn(&g, ws.get(), bytes, stream));
  return o;
}

void register_cache4(pybind11::module_& m) {
  m.def("cache4_plan", &cache4_plan, "pages, slots and positions of one step of a paged 4-bit cache");
  m.def("cache4_write", &cache4_write, "keys and values into the 4-bit cache");
  m.def("cache4_read", &cache4_read, "keys and values out of the 4-bit cache");
  m.def("attn_cache4", &attn_cache4, "attention against the paged 4-bit cache");
}
