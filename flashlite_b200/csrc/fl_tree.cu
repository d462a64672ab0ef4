// Attention of new tokens (one, a chunk, or a tree of drafted ones) over a
// paged cache: the plain kernel, one warp per (token, query head).
//
//   o_t = sum_j w_tj v_j / l_t,  w_tj = exp(scale q_t.k_j - m_t),
//   m_t = max_j, l_t = sum_j w_tj over the keys j that t sees:
//   the cached ones and the new ones its mask (or the causal rule) names.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "../../include/flashlite_b200.h"
#include "fl_internal.h"
#include "fl_ptx.cuh"

namespace fl {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxRequests = 4096;

struct TreeParams {
  fl_tree_attention_args a;
  float scale_log2;
  int page_shift;
  unsigned int* err;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) tree_attention_kernel(const __grid_constant__ TreeParams p) {
  const fl_tree_attention_args& a = p.a;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const long long w = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (w >= a.tokens * a.heads) return;
  const int t = static_cast<int>(w / a.heads), h = static_cast<int>(w % a.heads);
  const int kh = h / static_cast<int>(a.heads / a.kv_heads);
  int lo = 0, hi = static_cast<int>(a.requests);
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_seqlens[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int begin = a.cu_seqlens[lo], end = min(static_cast<long long>(a.cu_seqlens[lo + 1]), static_cast<long long>(a.tokens));
  const int i = t - begin, count = end - begin;
  constexpr int kPer = D / 32;
  float q[kPer], o[kPer];
  for (int e = 0; e < kPer; ++e) {
    q[e] = static_cast<float>(static_cast<const T*>(a.q)[t * a.q_stride[0] + h * a.q_stride[1] + lane + 32 * e]);
    o[e] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  if (begin >= 0 && i >= 0 && i < count) {
    const int ctx = a.context_lens[lo];
    long long keys = static_cast<long long>(ctx) + (a.tree_mask ? count : i + 1);
    const long long room = a.table_cols << p.page_shift;
    if (ctx < 0 || keys > room) {
      if (lane == 0) atomicOr(p.err, kDevErrIndex);
      keys = ctx < 0 ? 0 : room;
    }
    for (int j = 0; j < keys; ++j) {
      if (j >= ctx && a.tree_mask) {
        const int d = j - ctx;
        if (d >= 32 * a.mask_words || !((a.tree_mask[t * a.mask_words + (d >> 5)] >> (d & 31)) & 1)) continue;
      }
      const int block = a.block_table[lo * a.table_stride + (j >> p.page_shift)];
      if (block < 0 || block >= a.num_blocks) {
        if (lane == 0) atomicOr(p.err, kDevErrIndex);
        continue;
      }
      const int r = j & ((1 << p.page_shift) - 1);
      const T* kr = static_cast<const T*>(a.k_cache) + block * a.k_stride[0] + r * a.k_stride[1] + kh * a.k_stride[2];
      const T* vr = static_cast<const T*>(a.v_cache) + block * a.v_stride[0] + r * a.v_stride[1] + kh * a.v_stride[2];
      float s = 0.0f;
      for (int e = 0; e < kPer; ++e) s = fmaf(q[e], static_cast<float>(kr[lane + 32 * e]), s);
      for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s *= p.scale_log2;
      const float mn = fmaxf(m, s);
      const float alpha = (m == -INFINITY) ? 0.0f : ex2_approx(m - mn);
      const float w_ = (mn == -INFINITY) ? 0.0f : ex2_approx(s - mn);
      m = mn;
      l = l * alpha + w_;
      for (int e = 0; e < kPer; ++e) o[e] = o[e] * alpha + w_ * static_cast<float>(vr[lane + 32 * e]);
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : (l == l ? 0.0f : l);
  for (int e = 0; e < kPer; ++e)
    static_cast<T*>(a.out)[(static_cast<long long>(t) * a.heads + h) * D + lane + 32 * e] = static_cast<T>(o[e] * inv);
  if (a.lse && lane == 0) a.lse[static_cast<long long>(t) * a.heads + h] = l != 0.0f ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
}

int tree_attention(const fl_tree_attention_args* args, void* stream) {
  if (args == nullptr) return fail(FL_ERR_INVALID_ARGUMENT, "null argument block");
  const fl_tree_attention_args& a = *args;
  if (a.tokens < 0 || a.requests < 0 || a.heads < 0 || a.kv_heads < 0 || a.num_blocks < 0 || a.table_cols < 0 ||
      a.mask_words < 0)
    return fail(FL_ERR_INVALID_ARGUMENT, "negative size");
  if (a.head_dim != 64 && a.head_dim != 128)
    return fail(FL_ERR_UNSUPPORTED, "tree_attention requires head_dim 64 or 128");
  if (a.dtype != FL_DTYPE_F16 && a.dtype != FL_DTYPE_BF16)
    return fail(FL_ERR_UNSUPPORTED, "tree_attention supports fp16 and bf16");
  if (a.kv_heads == 0 ? a.heads != 0 : (a.heads % a.kv_heads != 0 || a.heads / a.kv_heads > 128))
    return fail(FL_ERR_INVALID_ARGUMENT, "heads must be a multiple of kv_heads, at most 128 times");
  if (a.page_size < 8 || a.page_size > 256 || (a.page_size & (a.page_size - 1)) != 0)
    return fail(FL_ERR_UNSUPPORTED, "page_size must be a power of two from 8 to 256");
  if (a.requests > kMaxRequests) return fail(FL_ERR_UNSUPPORTED, "at most 4096 requests");
  if (a.tokens > (1LL << 28) || a.heads > (1LL << 15) || a.num_blocks > 0x7fffffffLL || a.table_cols > (1LL << 26) ||
      a.mask_words > (1LL << 20))
    return fail(FL_ERR_INVALID_ARGUMENT, "dimension too large");
  if (a.tokens == 0 || a.heads == 0) return FL_OK;
  if (!a.q || !a.out || !a.cu_seqlens || (a.requests > 0 && !a.context_lens) ||
      (a.requests > 0 && a.table_cols > 0 && !a.block_table) || (a.num_blocks > 0 && (!a.k_cache || !a.v_cache)))
    return fail(FL_ERR_INVALID_ARGUMENT, "null tensor pointer");
  int st = check_device();
  if (st != FL_OK) return st;
  TreeParams p;
  p.a = a;
  p.err = device_error_word();
  double scale = a.sm_scale;
  if (scale == 0.0) scale = 1.0 / std::sqrt(static_cast<double>(a.head_dim));
  p.scale_log2 = static_cast<float>(scale * 1.44269504088896340736);
  p.page_shift = 0;
  while ((1LL << p.page_shift) < a.page_size) ++p.page_shift;
  const long long warps = a.tokens * a.heads;
  const int blocks = static_cast<int>((warps + kThreads / 32 - 1) / (kThreads / 32));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a.dtype == FL_DTYPE_F16)
    e = a.head_dim == 64 ? launch_pdl(tree_attention_kernel<__half, 64>, blocks, kThreads, 0, s, p)
                         : launch_pdl(tree_attention_kernel<__half, 128>, blocks, kThreads, 0, s, p);
  else
    e = a.head_dim == 64 ? launch_pdl(tree_attention_kernel<__nv_bfloat16, 64>, blocks, kThreads, 0, s, p)
                         : launch_pdl(tree_attention_kernel<__nv_bfloat16, 128>, blocks, kThreads, 0, s, p);
  return e == cudaSuccess ? FL_OK : cuda_fail(e, "tree attention launch");
}

}  // namespace
}  // namespace fl

extern "C" size_t fl_tree_attention_workspace_size(int64_t, int64_t, int64_t, int64_t) { return 0; }

extern "C" int fl_tree_attention(const fl_tree_attention_args* args, void* stream) {
  return fl::guarded([&] { return fl::tree_attention(args, stream); });
}
