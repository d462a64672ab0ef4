// Rotary positions: y = R(pos) x on the first `rot` of D columns of every
// head, the other columns copied. Pair j (0 <= j < rot/2) of a row at
// position p turns by the angle whose cosine and sine the table's row p
// holds: (x0, x1) -> (x0 c - x1 s, x1 c + x0 s), with x0, x1 the columns
// j, j + rot/2 (half layout) or 2j, 2j + 1 (interleaved). R is orthogonal up
// to the table's scale, so the gradient is the same with s negated
// (`inverse`). Products and sums are fp32, rounded once.
//
// The same kernel appends to a paged cache: rotated keys and unchanged values
// go to the rows that the slot map names instead of to k_out.
//
// Bound by memory: each element is read and written once. A lane owns 2 * VEC
// columns of a row (two 16-byte accesses) as A[VEC], B[VEC] of VEC pairs, and
// keeps their cosines and sines in registers while it walks over the heads,
// so the table is read once per token and warp, not once per head. The lanes
// of a warp that the columns of one row leave over take further heads where
// heads are closer together in memory than tokens, further tokens otherwise.

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

struct RotaryParams {
  fl_rotary_args a;
  unsigned int* err;
  int lanes;       // lanes per row: a power of two
  int units;       // (2 * VEC)-column units per row
  int rot_units;   // of which rotated
  int over_heads;  // what a warp's further lane groups take: heads (1) or tokens (0)
  int chunk;       // heads a warp walks over
  int n_chunks;
  int heads;       // q, k and v heads together
  long long warps; // warps with work
};

template <typename T>
__device__ __forceinline__ float to_f32(T x) { return static_cast<float>(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// One row's address: token (b, n) and head h of a tensor [B, N, H, D] given
// by its strides in elements.
template <typename T>
__device__ __forceinline__ long long row_of(const int64_t (&st)[3], long long b, long long n, int h) {
  return b * st[0] + n * st[1] + static_cast<long long>(h) * st[2];
}

template <typename T, int VEC, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long w = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (w >= p.warps) return;
  const fl_rotary_args& a = p.a;
  const int lane = threadIdx.x & 31;
  const int groups = 32 / p.lanes;
  const int g = lane / p.lanes;
  const int u0 = lane % p.lanes;
  const long long tokens = a.batch * a.length;
  const long long tw = w / p.n_chunks;
  const int h0 = static_cast<int>(w % p.n_chunks) * p.chunk;
  const int h1 = min(h0 + p.chunk, p.heads);
  const long long t = p.over_heads ? tw : tw * groups + g;
  if (t >= tokens) return;
  const int hstep = p.over_heads ? groups : 1;
  const long long b = t / a.length, n = t % a.length;

  const long long pi = (a.positions_batch ? t : n);
  const long long pos = a.positions == nullptr ? n
                        : a.positions_64 ? static_cast<const int64_t*>(a.positions)[pi]
                                         : static_cast<const int32_t*>(a.positions)[pi];
  const bool known = pos >= 0 && pos < a.table_rows;
  if (!known && u0 == 0 && p.err) atomicOr(p.err, kDevErrIndex);
  long long kc = 0, vc = 0;  // the token's row in the caches
  bool cached = false;
  if (a.slots != nullptr) {
    const long long slot = a.slots[t];
    cached = slot >= 0 && slot < a.cache_blocks * a.page_size;
    if (!cached && slot != -1 && u0 == 0 && p.err) atomicOr(p.err, kDevErrIndex);
    if (cached) {
      const long long blk = slot / a.page_size, r = slot % a.page_size;
      kc = blk * a.k_out_stride[0] + r * a.k_out_stride[1];
      vc = blk * a.v_out_stride[0] + r * a.v_out_stride[1];
    }
  }
  const int hq = static_cast<int>(a.heads), hk = static_cast<int>(a.kv_heads);

  for (int u = u0; u < p.units; u += p.lanes) {
    const bool turned = u < p.rot_units;
    // columns of A and B; in the scalar form an odd D leaves a unit without B
    const int ca = turned && !kInterleaved ? u * VEC : u * 2 * VEC;
    const int cb = turned && !kInterleaved ? static_cast<int>(a.rot / 2) + u * VEC : ca + VEC;
    const bool has_b = cb < a.head_dim;
    float c[VEC], s[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      c[j] = 1.0f;
      s[j] = 0.0f;
    }
    if (turned) {
      if (known) {
        const float* row = a.table + pos * a.rot;
        if constexpr (VEC >= 4) {
#pragma unroll
          for (int j = 0; j < VEC; j += 4) {
            const float4 cc = __ldg(reinterpret_cast<const float4*>(row + u * VEC + j));
            const float4 ss = __ldg(reinterpret_cast<const float4*>(row + a.rot / 2 + u * VEC + j));
            c[j] = cc.x; c[j + 1] = cc.y; c[j + 2] = cc.z; c[j + 3] = cc.w;
            s[j] = ss.x; s[j + 1] = ss.y; s[j + 2] = ss.z; s[j + 3] = ss.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            c[j] = row[u * VEC + j];
            s[j] = row[a.rot / 2 + u * VEC + j];
          }
        }
        if (a.inverse) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) s[j] = -s[j];
        }
      } else {  // a position outside the table: nothing to turn by, and not to be missed
#pragma unroll
        for (int j = 0; j < VEC; ++j) c[j] = s[j] = __int_as_float(0x7fc00000);
      }
    }
#pragma unroll 4
    for (int h = h0 + (p.over_heads ? g : 0); h < h1; h += hstep) {
      const T* src;
      T* dst;
      bool rotate = turned;
      if (h < hq) {
        src = static_cast<const T*>(a.q) + row_of<T>(a.q_stride, b, n, h);
        dst = static_cast<T*>(a.q_out) + row_of<T>(a.q_out_stride, b, n, h);
      } else if (h < hq + hk) {
        src = static_cast<const T*>(a.k) + row_of<T>(a.k_stride, b, n, h - hq);
        if (a.slots != nullptr) {
          if (!cached) continue;
          dst = static_cast<T*>(a.k_out) + kc + (h - hq) * a.k_out_stride[2];
        } else {
          dst = static_cast<T*>(a.k_out) + row_of<T>(a.k_out_stride, b, n, h - hq);
        }
      } else {
        if (!cached) continue;
        src = static_cast<const T*>(a.v) + row_of<T>(a.v_stride, b, n, h - hq - hk);
        dst = static_cast<T*>(a.v_out) + vc + (h - hq - hk) * a.v_out_stride[2];
        rotate = false;
      }
      Pack<T, VEC> x, y;
      x = *reinterpret_cast<const Pack<T, VEC>*>(src + ca);
      y = x;
      if (has_b) y = *reinterpret_cast<const Pack<T, VEC>*>(src + cb);
      if (rotate) {
        if constexpr (kInterleaved) {  // x, y hold 2 * VEC neighbouring columns: pairs (0,1), (2,3), ...
          T e[2 * VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            e[j] = x.v[j];
            e[VEC + j] = y.v[j];
          }
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float x0 = to_f32(e[2 * j]), x1 = to_f32(e[2 * j + 1]);
            e[2 * j] = from_f32<T>(fmaf(x0, c[j], -(x1 * s[j])));
            e[2 * j + 1] = from_f32<T>(fmaf(x1, c[j], x0 * s[j]));
          }
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            x.v[j] = e[j];
            y.v[j] = e[VEC + j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float x0 = to_f32(x.v[j]), x1 = to_f32(y.v[j]);
            x.v[j] = from_f32<T>(fmaf(x0, c[j], -(x1 * s[j])));
            y.v[j] = from_f32<T>(fmaf(x1, c[j], x0 * s[j]));
          }
        }
      }
      *reinterpret_cast<Pack<T, VEC>*>(dst + ca) = x;
      if (has_b) *reinterpret_cast<Pack<T, VEC>*>(dst + cb) = y;
    }
  }
}

bool aligned_for(const void* p, const int64_t (&st)[3], int vec) {
  return p == nullptr || (aligned16(p) && st[0] % vec == 0 && st[1] % vec == 0 && st[2] % vec == 0);
}

template <typename T, int VEC>
cudaError_t launch(const fl_rotary_args& a, cudaStream_t stream) {
  RotaryParams p;
  p.a = a;
  p.err = device_error_word();
  p.units = static_cast<int>((a.head_dim + 2 * VEC - 1) / (2 * VEC));
  p.rot_units = static_cast<int>(a.rot / (2 * VEC));
  p.lanes = 1;
  while (p.lanes < p.units && p.lanes < 32) p.lanes *= 2;
  const int groups = 32 / p.lanes;
  p.heads = static_cast<int>(a.heads + a.kv_heads * (a.v != nullptr ? 2 : 1));
  const int64_t(&near)[3] = a.heads > 0 ? a.q_stride : a.k_stride;
  p.over_heads = near[2] <= near[1] ? 1 : 0;
  const long long tokens = a.batch * a.length;
  const long long rows = p.over_heads ? tokens : (tokens + groups - 1) / groups;
  // A warp walks over all heads of its tokens where that leaves enough warps
  // to fill the GPU (16 per SM); with fewer tokens the heads are divided too.
  const int hstep = p.over_heads ? groups : 1;
  const int steps = (p.heads + hstep - 1) / hstep;
  const long long want = 16LL * sm_count();
  const long long split = std::min<long long>(steps, std::max<long long>(1, (want + rows - 1) / rows));
  p.chunk = static_cast<int>((steps + split - 1) / split) * hstep;
  p.n_chunks = (p.heads + p.chunk - 1) / p.chunk;
  p.warps = rows * p.n_chunks;
  const long long blocks = (p.warps + kThreads / 32 - 1) / (kThreads / 32);
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  return a.interleaved ? launch_pdl(rotary_kernel<T, VEC, true>, static_cast<int>(blocks), kThreads, 0, stream, p)
                       : launch_pdl(rotary_kernel<T, VEC, false>, static_cast<int>(blocks), kThreads, 0, stream, p);
}

template <typename T>
cudaError_t launch_typed(const fl_rotary_args& a, cudaStream_t stream) {
  // 16-byte accesses where pointers, strides and both halves of the rotated
  // columns allow them, single elements otherwise.
  constexpr int kVec = 16 / sizeof(T);
  const bool wide = a.head_dim % (2 * kVec) == 0 && a.rot % (2 * kVec) == 0 && aligned16(a.table) &&
                    aligned_for(a.q, a.q_stride, kVec) && aligned_for(a.q_out, a.q_out_stride, kVec) &&
                    aligned_for(a.k, a.k_stride, kVec) && aligned_for(a.k_out, a.k_out_stride, kVec) &&
                    aligned_for(a.v, a.v_stride, kVec) && aligned_for(a.v_out, a.v_out_stride, kVec);
  return wide ? launch<T, kVec>(a, stream) : launch<T, 1>(a, stream);
}

int rotary(const fl_rotary_args* args, void* stream) {
  if (args == nullptr) return fail(FL_ERR_INVALID_ARGUMENT, "null argument block");
  const fl_rotary_args& a = *args;
  if (a.batch < 0 || a.length < 0 || a.heads < 0 || a.kv_heads < 0 || a.table_rows < 0)
    return fail(FL_ERR_INVALID_ARGUMENT, "negative size");
  if (a.head_dim <= 0 || a.rot < 0 || a.rot > a.head_dim || a.rot % 2 != 0)
    return fail(FL_ERR_INVALID_ARGUMENT, "the rotated columns must be an even number up to head_dim");
  if (a.dtype != FL_DTYPE_F16 && a.dtype != FL_DTYPE_BF16 && a.dtype != FL_DTYPE_F32)
    return fail(FL_ERR_UNSUPPORTED, "rotary supports fp16, bf16 and fp32");
  if (a.length > (1LL << 30) || a.batch > (1LL << 30) || a.heads > (1LL << 16) || a.kv_heads > (1LL << 16) ||
      a.head_dim > (1LL << 16))
    return fail(FL_ERR_INVALID_ARGUMENT, "dimension too large");
  if (a.batch == 0 || a.length == 0 || a.heads + a.kv_heads == 0) return FL_OK;
  if ((a.heads > 0 && (!a.q || !a.q_out)) || (a.kv_heads > 0 && (!a.k || !a.k_out)) || (!a.table && a.rot > 0))
    return fail(FL_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if ((a.slots != nullptr) != (a.v != nullptr) || (a.v != nullptr && !a.v_out))
    return fail(FL_ERR_INVALID_ARGUMENT, "the cache form takes v, its cache and the slots together");
  if (a.slots != nullptr && (a.page_size <= 0 || a.cache_blocks < 0))
    return fail(FL_ERR_INVALID_ARGUMENT, "page_size must be positive");
  int st = check_device();
  if (st != FL_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a.dtype == FL_DTYPE_F16    ? launch_typed<__half>(a, s)
                        : a.dtype == FL_DTYPE_BF16 ? launch_typed<__nv_bfloat16>(a, s)
                                                   : launch_typed<float>(a, s);
  return e == cudaSuccess ? FL_OK : cuda_fail(e, "rotary launch");
}

}  // namespace
}  // namespace fl

extern "C" int fl_rotary(const fl_rotary_args* args, void* stream) {
  return fl::guarded([&] { return fl::rotary(args, stream); });
}
