// Bookkeeping of one serving step: block-table entries, slots and positions
// of the new tokens, ancestor masks of drafted trees.
//
//   have_b = max(held_b, ceil(ctx_b / page)), want_b = max(have_b, ceil((ctx_b + T_b) / page))
//   need_b = want_b - have_b (0 if the row is too short), upto = prefix sum
//   admitted_b = row long enough and (need_b == 0 or upto_b <= num_free)
//   block j of request b, have_b <= j < want_b:
//     free[num_free - 1 - (upto_b - need_b + j - have_b)]
//
// Bound by latency: a few bytes per request and token. One launch: every
// block computes the prefix sum over all requests again (8 bytes of shared
// memory per request) rather than a first kernel handing it to a second, and
// then serves its own share of the tokens (one thread each) and of the
// requests' table rows (one warp each). A token takes a fresh block's number
// from the free list itself, so no block waits for another's table entries.
// More than two blocks per SM pay for the sum too often (261,000 tokens of 509
// requests: 8.3 us with one, 6.7 with two, 9.2 with four).

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
constexpr int kMaxRequests = 16384;

struct PlanParams {
  fl_plan_args a;
  unsigned int* err;
};

struct Request {
  int begin, count, ctx, have, need;
  bool fits;
};

// A request's share of the arithmetic above. Lengths out of range count as
// none and are recorded; the request is refused and keeps the blocks it holds.
__device__ __forceinline__ Request request_from(const PlanParams& p, int ctx, int begin, int end, int held, bool report) {
  const fl_plan_args& a = p.a;
  Request r;
  r.ctx = ctx;
  r.begin = begin;
  const bool sound = r.ctx >= 0 && r.begin >= 0 && end >= r.begin && end <= a.tokens &&
                     r.ctx <= 0x7fffffff - (end - r.begin) - static_cast<int>(a.page_size);
  if (!sound) {
    if (report && p.err) atomicOr(p.err, kDevErrIndex);
    r.ctx = r.begin = r.count = r.need = 0;
    r.have = held;
    r.fits = false;
    return r;
  }
  r.count = end - r.begin;
  const int page = static_cast<int>(a.page_size);
  r.have = max(held, (r.ctx + page - 1) / page);
  const int want = max(r.have, (r.ctx + r.count + page - 1) / page);
  r.fits = want <= a.table_cols;
  r.need = r.fits ? want - r.have : 0;
  return r;
}
__device__ __forceinline__ Request request_of(const PlanParams& p, int b) {
  return request_from(p, p.a.context_lens[b], p.a.cu_seqlens[b], p.a.cu_seqlens[b + 1], p.a.held_blocks[b], false);
}

__global__ void __launch_bounds__(kThreads) plan_kernel(const __grid_constant__ PlanParams p) {
  extern __shared__ int smem[];
  const fl_plan_args& a = p.a;
  const int nb = static_cast<int>(a.requests), total = static_cast<int>(a.tokens);
  int* s_first = smem;    // [nb] blocks needed (-1: the row is too short), then taken by the requests before (-1: refused)
  int* s_cu = smem + nb;  // [nb] first token, rising
  __shared__ long long s_warp[kThreads / 32];
  __shared__ int s_used;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int page = static_cast<int>(a.page_size);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // This thread's first token's parent: on its way, with its neighbours', while
  // the requests are summed.
  const int t0 = blockIdx.x * kThreads + tid;
  int up0 = -1;
  if (a.parents != nullptr && t0 < total) up0 = a.parents[t0];
  // blocks that are not there cannot be given out
  const int free_n = max(0, min(a.num_free[0], static_cast<int>(a.free_capacity)));

  bool in_order = true;
  // ---- prefix sum of the blocks needed: each thread takes a run of requests ----
  constexpr int kAhead = 4;  // requests of a thread whose loads are under way together
  for (int base = tid; base < nb; base += kAhead * kThreads) {
    int ctx[kAhead], begin[kAhead], end[kAhead], held[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int b = min(base + i * kThreads, nb - 1);
      ctx[i] = a.context_lens[b];
      begin[i] = a.cu_seqlens[b];
      end[i] = a.cu_seqlens[b + 1];
      held[i] = a.held_blocks[b];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int b = base + i * kThreads;
      if (b >= nb) break;
      const Request r = request_from(p, ctx[i], begin[i], end[i], held[i], blockIdx.x == 0);
      s_first[b] = r.fits ? r.need : -1;
      const bool sound = begin[i] >= 0 && end[i] >= begin[i] && end[i] <= total;
      s_cu[b] = sound ? begin[i] : 0x7fffffff;
      in_order &= sound;
    }
  }
  if (tid == 0) s_used = 0;
  if (__syncthreads_or(!in_order)) {
    // Offsets out of range: those requests begin where the next sound one does,
    // so that the tokens' search below passes them by.
    if (tid == 0)
      for (int b = nb - 2; b >= 0; --b) s_cu[b] = min(s_cu[b], s_cu[b + 1]);
    __syncthreads();
  }
  const int per = (nb + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, nb), b1 = min(b0 + per, nb);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += max(s_first[b], 0);
  long long incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += x;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  long long upto = incl - mine;
  for (int w = 0; w < warp; ++w) upto += s_warp[w];
  int used = 0;
  for (int b = b0; b < b1; ++b) {
    const int need = s_first[b];
    const bool admitted = need == 0 || (need > 0 && upto + need <= free_n);
    s_first[b] = !admitted ? -1 : need > 0 ? static_cast<int>(upto) : 0;
    upto += max(need, 0);
    if (admitted && need > 0) used = static_cast<int>(upto);
  }
  if (blockIdx.x == 0 && used > 0) atomicMax(&s_used, used);
  __syncthreads();
  if (blockIdx.x == 0) {
    if (tid == 0) a.num_free_after[0] = free_n - s_used;
    for (int b = tid; b < nb; b += kThreads) a.admitted[b] = s_first[b] >= 0 ? 1 : 0;
  }
  // ---- table rows: one warp per request ----
  for (int b = blockIdx.x * (kThreads / 32) + warp; b < nb; b += gridDim.x * (kThreads / 32)) {
    const int first = s_first[b];
    const Request r = request_of(p, b);
    if (lane == 0) a.held_after[b] = r.have + (first >= 0 ? r.need : 0);
    if (first < 0) continue;
    int32_t* row = a.block_table + static_cast<int64_t>(b) * a.table_stride + r.have;
    for (int j = lane; j < r.need; j += 32) row[j] = a.free_blocks[free_n - 1 - first - j];
  }

  // ---- tokens: one thread each ----
  for (int t = t0; t < total; t += gridDim.x * kThreads) {
    int lo = 0, hi = nb;  // the last request that begins at or before t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_cu[mid] <= t) lo = mid;
      else hi = mid;
    }
    int64_t slot = -1;
    int pos = 0;
    const Request r = nb > 0 ? request_of(p, lo) : Request{0, 0, 0, 0, 0, false};
    const int i = t - r.begin;
    const bool inside = nb > 0 && i >= 0 && i < r.count;
    if (inside) {
      pos = r.ctx + i;
      const int first = s_first[lo];
      if (first >= 0) {
        const int j = pos / page;
        const int block = j < r.have ? a.block_table[static_cast<int64_t>(lo) * a.table_stride + j]
                                     : a.free_blocks[free_n - 1 - first - (j - r.have)];
        slot = static_cast<int64_t>(block) * page + pos % page;
      }
    }
    a.slots[t] = slot;
    if (a.parents != nullptr) {
      // Ancestors have falling indices: each mask word is complete when the
      // walk leaves it.
      uint32_t* row = a.tree_mask + static_cast<int64_t>(t) * a.mask_words;
      const int words = static_cast<int>(a.mask_words);
      int next = words - 1, depth = -1;  // next: highest word not yet written
      if (inside && i >= 32 * words) {
        if (p.err) atomicOr(p.err, kDevErrIndex);
      } else if (inside) {
        int node = i, word = i >> 5, up = t == t0 ? up0 : a.parents[t];
        uint32_t bits = 0;
        while (true) {
          if ((node >> 5) != word) {
            while (next > word) row[next--] = 0u;
            row[next--] = bits;
            word = node >> 5;
            bits = 0;
          }
          bits |= 1u << (node & 31);
          ++depth;
          if (up >= node || up < -1) {  // not a tree: taken as a root
            if (p.err) atomicOr(p.err, kDevErrIndex);
            break;
          }
          if (up < 0) break;
          node = up;
          up = a.parents[r.begin + node];
        }
        while (next > word) row[next--] = 0u;
        row[next--] = bits;
      }
      while (next >= 0) row[next--] = 0u;
      if (inside) pos = r.ctx + max(depth, 0);
    }
    a.positions[t] = pos;
  }
}

int plan(const fl_plan_args* args, void* stream) {
  if (args == nullptr) return fail(FL_ERR_INVALID_ARGUMENT, "null argument block");
  const fl_plan_args& a = *args;
  if (a.requests < 0 || a.tokens < 0 || a.table_cols < 0 || a.free_capacity < 0 || a.mask_words < 0)
    return fail(FL_ERR_INVALID_ARGUMENT, "negative size");
  if (a.page_size <= 0 || a.page_size > (1LL << 20))
    return fail(FL_ERR_INVALID_ARGUMENT, "page_size must be positive");
  if (a.requests > kMaxRequests) return fail(FL_ERR_UNSUPPORTED, "at most 16384 requests");
  if (a.tokens > (1LL << 30) || a.table_cols > (1LL << 30) || a.free_capacity > 0x7fffffffLL ||
      a.mask_words > (1LL << 20))
    return fail(FL_ERR_INVALID_ARGUMENT, "dimension too large");
  if (!a.cu_seqlens || !a.num_free || !a.num_free_after ||
      (a.requests > 0 && (!a.context_lens || !a.held_blocks || !a.admitted || !a.held_after || (a.table_cols > 0 && !a.block_table))) ||
      (a.free_capacity > 0 && !a.free_blocks) || (a.tokens > 0 && (!a.slots || !a.positions)))
    return fail(FL_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (a.parents != nullptr && a.tokens > 0 && (a.mask_words == 0 || !a.tree_mask))
    return fail(FL_ERR_INVALID_ARGUMENT, "a tree needs mask_words > 0 and a tree_mask");
  int st = check_device();
  if (st != FL_OK) return st;
  PlanParams p;
  p.a = a;
  p.err = device_error_word();
  const int smem = static_cast<int>(2 * a.requests) * 4;
  static std::atomic<bool> configured[kMaxFlagDevices];
  cudaError_t e = ensure_smem_limit(plan_kernel, 2 * kMaxRequests * 4, configured);
  if (e != cudaSuccess) return cuda_fail(e, "plan launch");
  const int64_t want = std::max<int64_t>((a.tokens + kThreads - 1) / kThreads,
                                         (a.requests + kThreads / 32 - 1) / (kThreads / 32));
  const int blocks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, 2 * sm_count())));
  e = launch_pdl(plan_kernel, blocks, kThreads, smem, static_cast<cudaStream_t>(stream), p);
  return e == cudaSuccess ? FL_OK : cuda_fail(e, "plan launch");
}

// A step's results into the state they follow, a thread for each request. A
// kernel of its own: every block of the first one reads all of the state.
struct SettleParams {
  const int32_t* context_lens;
  const uint8_t* admitted;
  const int32_t* held_after;
  const int32_t* num_free_after;
  int32_t* held_blocks;
  int32_t* num_free;
  int32_t* attention_lens;
  int requests;
};

__global__ void __launch_bounds__(kThreads) settle_kernel(const __grid_constant__ SettleParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = blockIdx.x * kThreads + threadIdx.x;
  if (b == 0) p.num_free[0] = p.num_free_after[0];
  if (b >= p.requests) return;
  p.held_blocks[b] = p.held_after[b];
  p.attention_lens[b] = p.admitted[b] ? p.context_lens[b] : -1;
}

int settle(const SettleParams& p, int64_t requests, void* stream) {
  if (requests < 0) return fail(FL_ERR_INVALID_ARGUMENT, "negative size");
  if (requests > kMaxRequests) return fail(FL_ERR_UNSUPPORTED, "at most 16384 requests");
  if (!p.num_free_after || !p.num_free ||
      (requests > 0 && (!p.context_lens || !p.admitted || !p.held_after || !p.held_blocks || !p.attention_lens)))
    return fail(FL_ERR_INVALID_ARGUMENT, "null tensor pointer");
  const int st = check_device();
  if (st != FL_OK) return st;
  const int blocks = std::max(1, (p.requests + kThreads - 1) / kThreads);
  const cudaError_t e = launch_pdl(settle_kernel, blocks, kThreads, 0, static_cast<cudaStream_t>(stream), p);
  return e == cudaSuccess ? FL_OK : cuda_fail(e, "settle launch");
}

}  // namespace
}  // namespace fl

extern "C" int fl_settle_step(const int32_t* context_lens, const uint8_t* admitted, const int32_t* held_after,
                              const int32_t* num_free_after, int32_t* held_blocks, int32_t* num_free,
                              int32_t* attention_lens, int64_t requests, void* stream) {
  return fl::guarded([&] {
    return fl::settle({context_lens, admitted, held_after, num_free_after, held_blocks, num_free, attention_lens,
                       static_cast<int>(requests)},
                      requests, stream);
  });
}

extern "C" int fl_plan_cache_step(const fl_plan_args* args, void* stream) {
  return fl::guarded([&] { return fl::plan(args, stream); });
}
