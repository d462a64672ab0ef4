// Torch binding of the serving entry points (rotary positions, cache step,
// attention over the paged cache). As in flash_attn.cpp, this file validates
// torch tensors, takes their strides and calls the C ABI
// (include/flashlite_b200.h); outputs and workspaces are torch allocations on
// the current stream of the tensors' device.

#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <tuple>

#include "../../include/flashlite_b200.h"

namespace {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

// Makes a call of the C ABI and turns its status into an error. The launch
// blocks while the device's launch queue is full; other Python threads keep
// running meanwhile (the error text is thread-local).
template <typename Call>
void launch(Call&& call) {
  int status;
  {
    pybind11::gil_scoped_release no_gil;
    status = call();
  }
  TORCH_CHECK(status == FL_OK, "flashlite_b200: ", fl_status_str(status), ": ", fl_last_error());
}

void* stream_of(const Tensor& t) {
  return static_cast<void*>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

// Outputs of a call: contiguous tensors one after the other in one allocation
// on the current stream of the current device, taken from torch's caching
// allocator directly. The calls of a serving step run for microseconds, and
// torch::empty costs most of one: six outputs 8.6 us a call, this way 5.3.
class Outputs {
 public:
  explicit Outputs(size_t bytes)
      : storage_(c10::Storage::use_byte_size_t(), bytes, c10::cuda::CUDACachingAllocator::get()->allocate(bytes),
                 c10::cuda::CUDACachingAllocator::get(), /*resizable=*/true) {}

  Tensor take(torch::IntArrayRef sizes, torch::ScalarType type) {
    const auto meta = c10::scalarTypeToTypeMeta(type);
    const size_t item = meta.itemsize();
    used_ = (used_ + item - 1) / item * item;
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(storage_),
                                                        c10::DispatchKeySet(c10::DispatchKey::CUDA), meta);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    t.unsafeGetTensorImpl()->set_storage_offset(static_cast<int64_t>(used_ / item));
    used_ += item * t.numel();
    TORCH_INTERNAL_ASSERT(used_ <= storage_.nbytes());
    return t;
  }

 private:
  c10::Storage storage_;
  size_t used_ = 0;
};

Tensor fresh(torch::IntArrayRef sizes, torch::ScalarType type) {
  size_t bytes = c10::elementSize(type);
  for (const int64_t n : sizes) bytes *= n;
  return Outputs(bytes).take(sizes, type);
}

// A tensor of the caller's that a call has written: torch is told, as by its own
// in-place operations, so that autograd finds a saved tensor changed. (Those of
// inference mode keep no version.)
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

bool given(const OptTensor& t) { return t.has_value() && t.value().defined(); }

int dtype_of(const Tensor& t, bool with_fp32, const char* who) {
  if (t.scalar_type() == torch::kHalf) return FL_DTYPE_F16;
  if (t.scalar_type() == torch::kBFloat16) return FL_DTYPE_BF16;
  if (with_fp32 && t.scalar_type() == torch::kFloat) return FL_DTYPE_F32;
  TORCH_CHECK(false, who, " supports fp16", with_fp32 ? ", bf16 and fp32" : " and bf16", " tensors");
}

void check_layout(const std::string& layout) {
  TORCH_CHECK(layout == "bhnd" || layout == "bnhd", "layout must be 'bhnd' or 'bnhd'");
}

// On q's device, innermost dimension contiguous.
void check_rows(const Tensor& t, const Tensor& q, const char* name) {
  TORCH_CHECK(t.is_cuda(), "All tensors must be on CUDA");
  TORCH_CHECK(t.device() == q.device(), "All tensors must be on the same CUDA device");
  TORCH_CHECK(t.size(-1) <= 1 || t.stride(-1) == 1, name, ": the last dimension must be contiguous");
}

// An output must not write one element twice.
void check_output(const Tensor& t, const char* name) {
  for (int64_t d = 0; d < t.dim(); ++d)
    TORCH_CHECK(t.size(d) <= 1 || t.stride(d) != 0, name, " must not be an expanded tensor");
}

// A contiguous vector (or matrix) of whole numbers on q's device.
void check_ints(const Tensor& t, const torch::Device& dev, torch::ScalarType type, int64_t dim, const char* name) {
  TORCH_CHECK(t.is_cuda(), "All tensors must be on CUDA");
  TORCH_CHECK(t.device() == dev, "All tensors must be on the same CUDA device");
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", torch::toString(type));
  TORCH_CHECK(t.dim() == dim, name, " must have ", dim, " dimension(s)");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

// Sizes and strides of [B, N, H, D] rows: 3-D tensors are [tokens, heads, D],
// 4-D ones follow `layout`.
struct Rows {
  int64_t batch, length, heads, dim;
  int64_t stride[3];
};

Rows rows_of(const Tensor& t, const std::string& layout) {
  Rows r;
  if (t.dim() == 3) {
    r = {1, t.size(0), t.size(1), t.size(2), {0, t.stride(0), t.stride(1)}};
  } else {
    const int n = layout == "bnhd" ? 1 : 2, h = 3 - n;
    r = {t.size(0), t.size(n), t.size(h), t.size(3), {t.stride(0), t.stride(n), t.stride(h)}};
  }
  return r;
}

void put(int64_t (&to)[3], const int64_t (&from)[3]) {
  for (int i = 0; i < 3; ++i) to[i] = from[i];
}

void set_positions(fl_rotary_args& a, const OptTensor& positions, const Tensor& q) {
  if (!given(positions)) return;
  const Tensor& p = positions.value();
  TORCH_CHECK(p.is_cuda() && p.device() == q.device(), "positions must be on q's CUDA device");
  TORCH_CHECK(p.scalar_type() == torch::kInt || p.scalar_type() == torch::kLong, "positions must be int32 or int64");
  TORCH_CHECK(p.is_contiguous(), "positions must be contiguous");
  const bool whole = p.dim() == 2 && p.size(0) == a.batch && p.size(1) == a.length;
  TORCH_CHECK(whole || (p.dim() == 1 && p.size(0) == a.length), "positions must be [N] or [B, N], one for each token");
  a.positions = p.data_ptr();
  a.positions_64 = p.scalar_type() == torch::kLong;
  a.positions_batch = whole;
}

void set_table(fl_rotary_args& a, const Tensor& table, const Tensor& q) {
  TORCH_CHECK(table.is_cuda() && table.device() == q.device(), "the table must be on q's CUDA device");
  TORCH_CHECK(table.scalar_type() == torch::kFloat && table.dim() == 2 && table.is_contiguous(),
              "the table must be a contiguous float32 matrix [positions, rotated columns]");
  TORCH_CHECK(table.size(1) % 2 == 0 && table.size(1) <= a.head_dim,
              "the table's columns must be an even number up to head_dim");
  a.table = table.data_ptr<float>();
  a.table_rows = table.size(0);
  a.rot = table.size(1);
}

Tensor output_like(const OptTensor& out, const Tensor& in, const char* name) {
  if (!given(out)) return fresh(in.sizes(), in.scalar_type());
  const Tensor& o = out.value();
  TORCH_CHECK(o.is_cuda() && o.device() == in.device(), name, " must be on the input's CUDA device");
  TORCH_CHECK(o.sizes() == in.sizes() && o.scalar_type() == in.scalar_type(), name, " must match its input");
  check_rows(o, in, name);
  check_output(o, name);
  return o;
}

// Rotary positions of q and (optionally) k, or their gradient.
std::tuple<Tensor, OptTensor> rotary_any(const Tensor& q, const OptTensor& k, const Tensor& table,
                                         const OptTensor& positions, bool interleaved, const std::string& layout,
                                         const OptTensor& out_q, const OptTensor& out_k, bool inverse) {
  check_layout(layout);
  TORCH_CHECK(q.is_cuda(), "All tensors must be on CUDA");
  TORCH_CHECK(q.dim() == 3 || q.dim() == 4, "q must be [tokens, heads, D] or 4D");
  check_rows(q, q, "q");
  const c10::cuda::CUDAGuard guard(q.device());
  fl_rotary_args a = {};
  a.dtype = dtype_of(q, true, "rotary");
  const Rows rq = rows_of(q, layout);
  a.batch = rq.batch;
  a.length = rq.length;
  a.heads = rq.heads;
  a.head_dim = rq.dim;
  put(a.q_stride, rq.stride);
  const Tensor oq = output_like(out_q, q, "out_q");
  put(a.q_out_stride, rows_of(oq, layout).stride);
  a.q = q.data_ptr();
  a.q_out = oq.data_ptr();
  OptTensor ok;
  if (given(k)) {
    const Tensor& kt = k.value();
    TORCH_CHECK(kt.dim() == q.dim() && kt.scalar_type() == q.scalar_type(), "k must have q's rank and type");
    check_rows(kt, q, "k");
    const Rows rk = rows_of(kt, layout);
    TORCH_CHECK(rk.batch == rq.batch && rk.length == rq.length && rk.dim == rq.dim,
                "k must match q in all but its heads");
    ok = output_like(out_k, kt, "out_k");
    a.kv_heads = rk.heads;
    put(a.k_stride, rk.stride);
    put(a.k_out_stride, rows_of(*ok, layout).stride);
    a.k = kt.data_ptr();
    a.k_out = ok->data_ptr();
  } else {
    TORCH_CHECK(!given(out_k), "out_k without k");
  }
  set_table(a, table, q);
  set_positions(a, positions, q);
  a.interleaved = interleaved;
  a.inverse = inverse;
  launch([&, stream = stream_of(q)] { return fl_rotary(&a, stream); });
  if (given(out_q)) written(oq);
  if (given(out_k)) written(*ok);
  return {oq, ok};
}

std::tuple<Tensor, OptTensor> rotary(const Tensor& q, const OptTensor& k, const Tensor& table,
                                     const OptTensor& positions, bool interleaved, const std::string& layout,
                                     const OptTensor& out_q, const OptTensor& out_k) {
  return rotary_any(q, k, table, positions, interleaved, layout, out_q, out_k, false);
}

std::tuple<Tensor, OptTensor> rotary_backward(const Tensor& dq, const OptTensor& dk, const Tensor& table,
                                              const OptTensor& positions, bool interleaved,
                                              const std::string& layout) {
  return rotary_any(dq, dk, table, positions, interleaved, layout, std::nullopt, std::nullopt, true);
}

// A cache [blocks, page, heads, D] ("bnhd") or [blocks, heads, page, D] ("bhnd").
Rows cache_of(const Tensor& c, const Tensor& q, const std::string& layout, const char* name) {
  TORCH_CHECK(c.dim() == 4, name,
              layout == "bnhd" ? " must be 4D [blocks, page, heads, D]" : " must be 4D [blocks, heads, page, D]");
  TORCH_CHECK(c.scalar_type() == q.scalar_type(), name, " must have q's type");
  check_rows(c, q, name);
  return rows_of(c, layout);
}

// Rotates q and k and writes k and v to their slots of the cache.
Tensor rotary_append(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table,
                     const OptTensor& positions, const Tensor& slots, const Tensor& k_cache, const Tensor& v_cache,
                     bool interleaved, const std::string& layout, const OptTensor& out_q) {
  check_layout(layout);
  TORCH_CHECK(q.is_cuda(), "All tensors must be on CUDA");
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "q, k and v must be [tokens, heads, D]");
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "k and v must have q's type");
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(2) == q.size(2) && v.sizes() == k.sizes(),
              "k and v must match q in all but their heads");
  check_rows(q, q, "q");
  check_rows(k, q, "k");
  check_rows(v, q, "v");
  check_ints(slots, q.device(), torch::kLong, 1, "slots");
  TORCH_CHECK(slots.size(0) == q.size(0), "slots must hold one slot for each token");
  const c10::cuda::CUDAGuard guard(q.device());
  fl_rotary_args a = {};
  a.dtype = dtype_of(q, true, "rotary_append");
  a.batch = 1;
  a.length = q.size(0);
  a.heads = q.size(1);
  a.kv_heads = k.size(1);
  a.head_dim = q.size(2);
  const Rows ck = cache_of(k_cache, q, layout, "k_cache"), cv = cache_of(v_cache, q, layout, "v_cache");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes(), "k_cache and v_cache must have the same shape");
  TORCH_CHECK(ck.heads == k.size(1) && ck.dim == q.size(2), "the caches must have k's heads and head_dim");
  check_output(k_cache, "k_cache");
  check_output(v_cache, "v_cache");
  const Tensor oq = output_like(out_q, q, "out_q");
  put(a.q_stride, rows_of(q, layout).stride);
  put(a.k_stride, rows_of(k, layout).stride);
  put(a.v_stride, rows_of(v, layout).stride);
  put(a.q_out_stride, rows_of(oq, layout).stride);
  put(a.k_out_stride, ck.stride);
  put(a.v_out_stride, cv.stride);
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.q_out = oq.data_ptr();
  a.k_out = k_cache.data_ptr();
  a.v_out = v_cache.data_ptr();
  a.slots = slots.data_ptr<int64_t>();
  a.cache_blocks = ck.batch;
  a.page_size = ck.length;
  set_table(a, table, q);
  set_positions(a, positions, q);
  a.interleaved = interleaved;
  if (a.length == 0) return oq;
  launch([&, stream = stream_of(q)] { return fl_rotary(&a, stream); });
  written(k_cache);
  written(v_cache);
  if (given(out_q)) written(oq);
  return oq;
}

// Blocks, slots, positions and tree masks of one serving step.
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, OptTensor> plan_cache_step(
    const Tensor& context_lens, const Tensor& cu_seqlens, const Tensor& block_table, const Tensor& held_blocks,
    const Tensor& free_blocks, const Tensor& num_free, int64_t total_tokens, int64_t page_size, const OptTensor& parents,
    int64_t mask_words) {
  TORCH_CHECK(context_lens.is_cuda(), "All tensors must be on CUDA");
  const torch::Device dev = context_lens.device();
  check_ints(context_lens, dev, torch::kInt, 1, "context_lens");
  check_ints(cu_seqlens, dev, torch::kInt, 1, "cu_seqlens");
  check_ints(held_blocks, dev, torch::kInt, 1, "held_blocks");
  check_ints(free_blocks, dev, torch::kInt, 1, "free_blocks");
  check_ints(num_free, dev, torch::kInt, 1, "num_free");
  TORCH_CHECK(block_table.is_cuda() && block_table.device() == dev, "All tensors must be on the same CUDA device");
  TORCH_CHECK(block_table.scalar_type() == torch::kInt && block_table.dim() == 2, "block_table must be an Int matrix");
  TORCH_CHECK(block_table.size(1) <= 1 || block_table.stride(1) == 1, "block_table: the last dimension must be contiguous");
  check_output(block_table, "block_table");
  const int64_t n = context_lens.size(0);
  TORCH_CHECK(cu_seqlens.size(0) == n + 1, "cu_seqlens must hold one value more than context_lens");
  TORCH_CHECK(block_table.size(0) == n, "block_table must have a row for each request");
  TORCH_CHECK(held_blocks.size(0) == n, "held_blocks must hold one value for each request");
  TORCH_CHECK(num_free.size(0) == 1, "num_free must hold one value");
  TORCH_CHECK(total_tokens >= 0 && mask_words >= 0, "total_tokens and mask_words must not be negative");
  const c10::cuda::CUDAGuard guard(dev);
  fl_plan_args a = {};
  OptTensor mask;
  if (given(parents)) {
    check_ints(parents.value(), dev, torch::kInt, 1, "parents");
    TORCH_CHECK(parents->size(0) == total_tokens, "parents must hold one value for each token");
    TORCH_CHECK(mask_words > 0, "a tree needs mask_words > 0");
    a.parents = parents->data_ptr<int32_t>();
  }
  // What belongs to the step, and what the cache keeps after it.
  Outputs step(static_cast<size_t>(total_tokens) * (12 + (a.parents ? 4 * mask_words : 0)) + n), kept(4 * (n + 1));
  Tensor slots = step.take({total_tokens}, torch::kLong);
  Tensor positions = step.take({total_tokens}, torch::kInt);
  if (a.parents != nullptr) {
    mask = step.take({total_tokens, mask_words}, torch::kInt);
    a.tree_mask = reinterpret_cast<uint32_t*>(mask->data_ptr<int32_t>());
  }
  Tensor admitted = step.take({n}, torch::kBool);
  Tensor left = kept.take({1}, torch::kInt), held = kept.take({n}, torch::kInt);
  a.context_lens = context_lens.data_ptr<int32_t>();
  a.cu_seqlens = cu_seqlens.data_ptr<int32_t>();
  a.block_table = block_table.data_ptr<int32_t>();
  a.held_blocks = held_blocks.data_ptr<int32_t>();
  a.held_after = held.data_ptr<int32_t>();
  a.free_blocks = free_blocks.data_ptr<int32_t>();
  a.num_free = num_free.data_ptr<int32_t>();
  a.slots = slots.data_ptr<int64_t>();
  a.positions = positions.data_ptr<int32_t>();
  a.admitted = reinterpret_cast<uint8_t*>(admitted.data_ptr<bool>());
  a.num_free_after = left.data_ptr<int32_t>();
  a.requests = n;
  a.tokens = total_tokens;
  a.table_cols = block_table.size(1);
  a.table_stride = block_table.stride(0);
  a.free_capacity = free_blocks.size(0);
  a.page_size = page_size;
  a.mask_words = mask_words;
  launch([&, stream = stream_of(context_lens)] { return fl_plan_cache_step(&a, stream); });
  written(block_table);
  return {slots, positions, admitted, left, held, mask};
}

// A step's held blocks and free count into the state that they follow; returns
// the lengths that attention takes.
Tensor settle_step(const Tensor& context_lens, const Tensor& held_blocks, const Tensor& num_free, const Tensor& admitted,
                   const Tensor& held_after, const Tensor& free_after) {
  TORCH_CHECK(context_lens.is_cuda(), "All tensors must be on CUDA");
  const torch::Device dev = context_lens.device();
  const int64_t n = context_lens.size(0);
  check_ints(context_lens, dev, torch::kInt, 1, "context_lens");
  check_ints(held_blocks, dev, torch::kInt, 1, "held_blocks");
  check_ints(num_free, dev, torch::kInt, 1, "num_free");
  check_ints(admitted, dev, torch::kBool, 1, "admitted");
  check_ints(held_after, dev, torch::kInt, 1, "held_after");
  check_ints(free_after, dev, torch::kInt, 1, "free_after");
  TORCH_CHECK(held_blocks.size(0) == n && admitted.size(0) == n && held_after.size(0) == n,
              "held_blocks, admitted and held_after must hold one value for each request");
  TORCH_CHECK(num_free.size(0) == 1 && free_after.size(0) == 1, "num_free and free_after must hold one value");
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor lens = fresh({n}, torch::kInt);
  launch([&, stream = stream_of(context_lens)] {
    return fl_settle_step(context_lens.data_ptr<int32_t>(), reinterpret_cast<const uint8_t*>(admitted.data_ptr<bool>()),
                          held_after.data_ptr<int32_t>(), free_after.data_ptr<int32_t>(), held_blocks.data_ptr<int32_t>(),
                          num_free.data_ptr<int32_t>(), lens.data_ptr<int32_t>(), n, stream);
  });
  written(held_blocks);
  written(num_free);
  return lens;
}

// Attention of new tokens over the paged cache. Returns (out, lse).
std::tuple<Tensor, OptTensor> tree_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                                             const Tensor& block_table, const Tensor& context_lens,
                                             const Tensor& cu_seqlens, const OptTensor& tree_mask, double sm_scale,
                                             const std::string& layout, const OptTensor& out, bool return_lse) {
  check_layout(layout);
  TORCH_CHECK(q.is_cuda(), "All tensors must be on CUDA");
  TORCH_CHECK(q.dim() == 3, "q must be [tokens, heads, D]");
  check_rows(q, q, "q");
  fl_tree_attention_args a = {};
  a.dtype = dtype_of(q, false, "tree_attention");
  const Rows ck = cache_of(k_cache, q, layout, "k_cache"), cv = cache_of(v_cache, q, layout, "v_cache");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes(), "k_cache and v_cache must have the same shape");
  TORCH_CHECK(ck.dim == q.size(2), "the caches must have q's head_dim");
  check_ints(context_lens, q.device(), torch::kInt, 1, "context_lens");
  check_ints(cu_seqlens, q.device(), torch::kInt, 1, "cu_seqlens");
  TORCH_CHECK(block_table.is_cuda() && block_table.device() == q.device(),
              "All tensors must be on the same CUDA device");
  TORCH_CHECK(block_table.scalar_type() == torch::kInt && block_table.dim() == 2, "block_table must be an Int matrix");
  TORCH_CHECK(block_table.size(1) <= 1 || block_table.stride(1) == 1, "block_table: the last dimension must be contiguous");
  a.requests = context_lens.size(0);
  TORCH_CHECK(cu_seqlens.size(0) == a.requests + 1, "cu_seqlens must hold one value more than context_lens");
  TORCH_CHECK(block_table.size(0) == a.requests, "block_table must have a row for each request");
  a.tokens = q.size(0);
  a.heads = q.size(1);
  a.head_dim = q.size(2);
  a.kv_heads = ck.heads;
  if (given(tree_mask)) {
    check_ints(tree_mask.value(), q.device(), torch::kInt, 2, "tree_mask");
    TORCH_CHECK(tree_mask->size(0) == a.tokens && tree_mask->size(1) > 0, "tree_mask must be [tokens, words]");
    a.tree_mask = reinterpret_cast<const uint32_t*>(tree_mask->data_ptr<int32_t>());
    a.mask_words = tree_mask->size(1);
  }
  const c10::cuda::CUDAGuard guard(q.device());
  Tensor out_tensor;
  if (given(out)) {
    out_tensor = out.value();
    TORCH_CHECK(out_tensor.is_cuda() && out_tensor.is_contiguous(), "out tensor must be contiguous CUDA tensor");
    TORCH_CHECK(out_tensor.sizes() == q.sizes(), "out tensor shape must match q");
    TORCH_CHECK(out_tensor.scalar_type() == q.scalar_type(), "out tensor must have q's type");
    TORCH_CHECK(out_tensor.device() == q.device(), "out tensor must be on the same device as q");
  } else {
    out_tensor = fresh(q.sizes(), q.scalar_type());
  }
  OptTensor lse;
  if (return_lse) {
    lse = fresh({a.tokens, a.heads}, torch::kFloat);
    a.lse = lse->data_ptr<float>();
  }
  const size_t bytes = fl_tree_attention_workspace_size(a.tokens, a.heads, a.kv_heads, a.head_dim);
  const c10::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
  a.workspace = ws.get();
  a.workspace_bytes = bytes;
  a.q = q.data_ptr();
  a.k_cache = k_cache.data_ptr();
  a.v_cache = v_cache.data_ptr();
  a.out = out_tensor.data_ptr();
  a.block_table = block_table.data_ptr<int32_t>();
  a.context_lens = context_lens.data_ptr<int32_t>();
  a.cu_seqlens = cu_seqlens.data_ptr<int32_t>();
  a.num_blocks = ck.batch;
  a.page_size = ck.length;
  a.table_cols = block_table.size(1);
  a.table_stride = block_table.stride(0);
  a.q_stride[0] = q.stride(0);
  a.q_stride[1] = q.stride(1);
  put(a.k_stride, ck.stride);
  put(a.v_stride, cv.stride);
  a.sm_scale = static_cast<float>(sm_scale);
  launch([&, stream = stream_of(q)] { return fl_tree_attention(&a, stream); });
  if (given(out)) written(out_tensor);
  return {out_tensor, lse};
}

}  // namespace

void bind_serving(pybind11::module_& m) {
  m.def("rotary", &rotary, "Rotary positions of q and k; returns (q, k)", py::arg("q"), py::arg("k"),
        py::arg("table"), py::arg("positions") = py::none(), py::arg("interleaved") = false,
        py::arg("layout") = "bnhd", py::arg("out_q") = py::none(), py::arg("out_k") = py::none());
  m.def("rotary_backward", &rotary_backward, "Gradient of rotary; returns (dq, dk)", py::arg("dq"), py::arg("dk"),
        py::arg("table"), py::arg("positions") = py::none(), py::arg("interleaved") = false,
        py::arg("layout") = "bnhd");
  m.def("rotary_append", &rotary_append, "Rotate q and k, write k and v to their cache slots; returns q",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("table"), py::arg("positions"), py::arg("slots"),
        py::arg("k_cache"), py::arg("v_cache"), py::arg("interleaved") = false, py::arg("layout") = "bnhd",
        py::arg("out_q") = py::none());
  m.def("plan_cache_step", &plan_cache_step,
        "Block table, slots and positions of one serving step; returns (slots, positions, admitted, num_free, held_blocks, tree_mask)",
        py::arg("context_lens"), py::arg("cu_seqlens"), py::arg("block_table"), py::arg("held_blocks"), py::arg("free_blocks"),
        py::arg("num_free"), py::arg("total_tokens"), py::arg("page_size"), py::arg("parents") = py::none(),
        py::arg("mask_words") = 0);
  m.def("settle_step", &settle_step,
        "Held blocks and free count of a step into the cache's state; returns the lengths that attention takes",
        py::arg("context_lens"), py::arg("held_blocks"), py::arg("num_free"), py::arg("admitted"), py::arg("held_after"),
        py::arg("free_after"));
  m.def("tree_attention", &tree_attention, "Attention of new tokens over a paged cache; returns (out, lse)",
        py::arg("q"), py::arg("k_cache"), py::arg("v_cache"), py::arg("block_table"), py::arg("context_lens"),
        py::arg("cu_seqlens"), py::arg("tree_mask") = py::none(), py::arg("sm_scale") = 0.0,
        py::arg("layout") = "bnhd", py::arg("out") = py::none(), py::arg("return_lse") = false);
}
