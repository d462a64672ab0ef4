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
// Bound by memory: each element is read and written once. A lane owns two
// 16-byte vectors of a row and walks over a token's heads with their cosines
// and sines in registers, so the table is read once per token and warp, not
// once per head. The lanes of a warp that the columns of one row leave over
// take further heads where heads are closer together in memory than tokens and
// many enough, further tokens otherwise. What it takes is bytes under way: through
// registers, two heads at a time at 24 warps per SM, a training step's q and
// k of 1 GB ran at 5.1 TB/s; with asynchronous copies into slots of shared
// memory that are each thread's own, four heads ahead, at 6.6 TB/s (153 us
// for 3 x 16381 tokens of 32 + 8 heads of 128, bf16; a copy of as many bytes
// 154 us), 8191 tokens of 32 + 8 + 8 heads appended to a cache 58 -> 36 us.
// Interleaved pairs need whole vectors side by side across the lanes: with
// both vectors of a lane side by side, each access used half of each sector
// (223 us for the 153).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <type_traits>

#include "../../include/flashlite_b200.h"
#include "fl_internal.h"
#include "fl_ptx.cuh"
#include "fl_types.cuh"

namespace fl {
namespace {

constexpr int kThreads = 256;

// Heads of a lane under way, and blocks per SM: 4 x 32 bytes x 768 threads =
// 96 KB per SM. Depths of 3 and 8, and 4 blocks (fewer registers), measured
// within 5 % of it over the sizes below.
constexpr int kDepth = 4;
constexpr int kBlocksPerSm = 3;
constexpr int kManyWaves = 8, kMaxDivision = 64;

struct RotaryParams {
  fl_rotary_args a;
  unsigned int* err;
  int lanes;       // lanes per row: a power of two
  int units;       // units of two vectors per row
  int rot_units;   // of which rotated (half layout)
  int over_heads;  // what a warp's further lane groups take: heads (1) or tokens (0)
  int heads;       // q, k and v heads together
  int chunk;       // of which a warp takes so many
  uint32_t n_chunks, tokens, length, warps;  // chunks; warps with work
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// Asynchronous 16-byte copy to shared memory, past L1.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Turns pairs. Half layout: x has the first column of VEC pairs and y the
// second. Interleaved: x and y hold VEC / 2 pairs each, (0, 1), (2, 3), ...,
// turned if tx, ty; the angles of y's pairs follow those of x's. (Single
// elements, VEC = 1, are one pair either way.) 16-bit types go through
// registers two elements at a time.
template <typename T, int VEC, bool kInterleaved>
__device__ __forceinline__ void turn(Pack<T, VEC>& x, Pack<T, VEC>& y, const float (&c)[VEC], const float (&s)[VEC],
                                     bool tx, bool ty) {
  if constexpr (VEC == 8) {
    uint32_t* xw = reinterpret_cast<uint32_t*>(&x);
    uint32_t* yw = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 e = unpack2<T>(xw[j]), f = unpack2<T>(yw[j]);
      if constexpr (kInterleaved) {
        if (tx) xw[j] = pack2<T>(fmaf(e.x, c[j], -(e.y * s[j])), fmaf(e.y, c[j], e.x * s[j]));
        if (ty) yw[j] = pack2<T>(fmaf(f.x, c[j + 4], -(f.y * s[j + 4])), fmaf(f.y, c[j + 4], f.x * s[j + 4]));
      } else if (tx) {
        xw[j] = pack2<T>(fmaf(e.x, c[2 * j], -(f.x * s[2 * j])), fmaf(e.y, c[2 * j + 1], -(f.y * s[2 * j + 1])));
        yw[j] = pack2<T>(fmaf(f.x, c[2 * j], e.x * s[2 * j]), fmaf(f.y, c[2 * j + 1], e.y * s[2 * j + 1]));
      }
    }
  } else if constexpr (kInterleaved && VEC > 1) {
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) {
      const float x0 = x.v[2 * j], x1 = x.v[2 * j + 1], y0 = y.v[2 * j], y1 = y.v[2 * j + 1];
      if (tx) {
        x.v[2 * j] = fmaf(x0, c[j], -(x1 * s[j]));
        x.v[2 * j + 1] = fmaf(x1, c[j], x0 * s[j]);
      }
      if (ty) {
        y.v[2 * j] = fmaf(y0, c[VEC / 2 + j], -(y1 * s[VEC / 2 + j]));
        y.v[2 * j + 1] = fmaf(y1, c[VEC / 2 + j], y0 * s[VEC / 2 + j]);
      }
    }
  } else if (tx) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float x0 = static_cast<float>(x.v[j]), x1 = static_cast<float>(y.v[j]);
      x.v[j] = static_cast<T>(fmaf(x0, c[j], -(x1 * s[j])));
      y.v[j] = static_cast<T>(fmaf(x1, c[j], x0 * s[j]));
    }
  }
}

// One row's address: token (b, n) and head h of a tensor [B, N, H, D] given
// by its strides in elements.
__device__ __forceinline__ long long row_of(const int64_t (&st)[3], long long b, long long n, int h) {
  return b * st[0] + n * st[1] + static_cast<long long>(h) * st[2];
}

template <typename T, int VEC, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) rotary_kernel(const __grid_constant__ RotaryParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t w = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (w >= p.warps) return;
  const fl_rotary_args& a = p.a;
  const int lane = threadIdx.x & 31;
  const int groups = 32 / p.lanes;
  const int g = lane / p.lanes, u0 = lane % p.lanes;
  const uint32_t tw = w / p.n_chunks, chunk = w - tw * p.n_chunks;
  const uint32_t t = p.over_heads ? tw : tw * groups + g;
  if (t >= p.tokens) return;
  const uint32_t b = t / p.length, n = t - b * p.length;
  const int hstep = p.over_heads ? groups : 1;
  const int hq = static_cast<int>(a.heads), hk = static_cast<int>(a.kv_heads);
  const int h0 = chunk * p.chunk;
  const T* q_in = static_cast<const T*>(a.q) + row_of(a.q_stride, b, n, 0);
  const T* k_in = static_cast<const T*>(a.k) + row_of(a.k_stride, b, n, 0);
  const T* v_in = static_cast<const T*>(a.v) + row_of(a.v_stride, b, n, 0);
  T* q_out = static_cast<T*>(a.q_out) + row_of(a.q_out_stride, b, n, 0);
  asm volatile("griddepcontrol.wait;" ::: "memory");

  const uint32_t pi = a.positions_batch ? t : n;
  const long long pos = a.positions == nullptr ? n
                        : a.positions_64 ? static_cast<const int64_t*>(a.positions)[pi]
                                         : static_cast<const int32_t*>(a.positions)[pi];
  const bool known = pos >= 0 && pos < a.table_rows;
  long long kc = 0, vc = 0;  // the token's row in the caches
  bool cached = false;
  bool sound = known || a.rot == 0;
  if (a.slots != nullptr) {
    const long long slot = a.slots[t];
    cached = slot >= 0 && slot < a.cache_blocks * a.page_size;
    if (cached) {
      const long long blk = ((slot | a.page_size) >> 32) == 0
                                ? static_cast<uint32_t>(slot) / static_cast<uint32_t>(a.page_size)
                                : slot / a.page_size;
      const long long r = slot - blk * a.page_size;
      kc = blk * a.k_out_stride[0] + r * a.k_out_stride[1];
      vc = blk * a.v_out_stride[0] + r * a.v_out_stride[1];
    } else {
      // a token that the cache step refused: its position may be anywhere
      sound = slot == -1;
    }
  }
  if (!sound && u0 == 0 && p.err) atomicOr(p.err, kDevErrIndex);

  T* k_out = static_cast<T*>(a.k_out) + (a.slots == nullptr ? row_of(a.k_out_stride, b, n, 0) : kc);
  T* v_out = static_cast<T*>(a.v_out) + vc;
  // a token without a slot has only its q heads
  const int last = min(h0 + p.chunk, a.slots == nullptr || cached ? p.heads : hq);

  for (int u = u0; u < p.units; u += p.lanes) {
    // The unit's two vectors A and B: neighbouring lanes take neighbouring
    // vectors, so that each access of a warp covers whole sectors.
    const int rot = static_cast<int>(a.rot), dim = static_cast<int>(a.head_dim);
    int ca, cb;
    if (VEC > 1 && kInterleaved) {
      ca = u * VEC;
      cb = dim / 2 + ca;
    } else if (kInterleaved) {
      ca = 2 * u;
      cb = ca + 1;
    } else if (u < p.rot_units) {
      ca = u * VEC;
      cb = rot / 2 + ca;
    } else {  // columns that are copied
      const int left = (dim - rot + 2 * VEC - 1) / (2 * VEC);
      ca = rot + (u - p.rot_units) * VEC;
      cb = ca + left * VEC;
    }
    const bool has_b = cb < dim;  // single elements: an odd number of copied columns leaves one without
    const bool turn_a = ca < rot, turn_b = cb < rot;
    float c[VEC], s[VEC];
    auto angles = [&] {
#pragma unroll
      for (int j = 0; j < VEC; ++j) c[j] = s[j] = __int_as_float(0x7fc00000);
      if (!known) return;  // a position outside the table leaves NaN: nothing to turn by, and not to be missed
      const float* row = a.table + pos * a.rot;
      auto get = [&](int pair, int j, auto count) {  // the angles of `count` pairs into c[j], s[j] on
        constexpr int kCount = decltype(count)::value;
        if constexpr (kCount % 4 == 0) {
#pragma unroll
          for (int e = 0; e < kCount; e += 4) {
            const float4 cc = __ldg(reinterpret_cast<const float4*>(row + pair + e));
            const float4 ss = __ldg(reinterpret_cast<const float4*>(row + rot / 2 + pair + e));
            c[j + e] = cc.x; c[j + e + 1] = cc.y; c[j + e + 2] = cc.z; c[j + e + 3] = cc.w;
            s[j + e] = ss.x; s[j + e + 1] = ss.y; s[j + e + 2] = ss.z; s[j + e + 3] = ss.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < kCount; ++e) {
            c[j + e] = row[pair + e];
            s[j + e] = row[rot / 2 + pair + e];
          }
        }
      };
      if constexpr (VEC > 1 && kInterleaved) {
        if (turn_a) get(ca / 2, 0, std::integral_constant<int, VEC / 2>{});
        if (turn_b) get(cb / 2, VEC / 2, std::integral_constant<int, VEC / 2>{});
      } else if (turn_a) {
        get(u * VEC, 0, std::integral_constant<int, VEC>{});
      }
      if (a.inverse) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[j] = -s[j];
      }
    };
    // The lane's heads one after the other: head `it` of q, then k, then v.
    const int first = h0 + (p.over_heads ? g : 0);
    struct Place {
      const T* src;
      T* dst;
      bool rotated;  // not v
    };
    auto place = [&](int h) -> Place {
      if (h < hq) return {q_in + h * a.q_stride[2], q_out + h * a.q_out_stride[2], true};
      h -= hq;
      if (h < hk) return {k_in + h * a.k_stride[2], k_out + h * a.k_out_stride[2], true};
      h -= hk;
      return {v_in + h * a.v_stride[2], v_out + h * a.v_out_stride[2], false};
    };
    if constexpr (VEC * sizeof(T) == 16) {
      // kDepth heads are under way in slots of shared memory that are this
      // thread's own, so no barrier is needed. (Outputs may be the inputs:
      // no element is anyone else's.)
      extern __shared__ __align__(16) uint4 slots[];
      const uint32_t mine = smem_u32(slots + threadIdx.x);
      auto fetch = [&](int h, int i) {
        if (h < last) {
          const T* src = place(h).src;
          copy16(mine + (2 * i) * (kThreads * 16), src + ca);
          copy16(mine + (2 * i + 1) * (kThreads * 16), src + cb);
        }
        copy_commit();
      };
#pragma unroll
      for (int i = 0; i < kDepth; ++i) fetch(first + i * hstep, i);
      angles();
      int i = 0;
#pragma unroll 1
      for (int h = first; h < last; h += hstep) {
        copy_wait<kDepth - 1>();
        Pack<T, VEC> x, y;
        *reinterpret_cast<uint4*>(&x) = slots[(2 * i) * kThreads + threadIdx.x];
        *reinterpret_cast<uint4*>(&y) = slots[(2 * i + 1) * kThreads + threadIdx.x];
        const Place at = place(h);
        if (at.rotated) turn<T, VEC, kInterleaved>(x, y, c, s, turn_a, turn_b);
        *reinterpret_cast<uint4*>(at.dst + ca) = *reinterpret_cast<const uint4*>(&x);
        *reinterpret_cast<uint4*>(at.dst + cb) = *reinterpret_cast<const uint4*>(&y);
        fetch(h + kDepth * hstep, i);
        i = i + 1 == kDepth ? 0 : i + 1;
      }
      copy_wait<0>();
    } else {
      angles();
      for (int h = first; h < last; h += hstep) {
        const Place at = place(h);
        Pack<T, VEC> x, y;
        x.v[0] = at.src[ca];
        y.v[0] = x.v[0];
        if (has_b) y.v[0] = at.src[cb];
        if (at.rotated) turn<T, VEC, kInterleaved>(x, y, c, s, turn_a, turn_b);
        at.dst[ca] = x.v[0];
        if (has_b) at.dst[cb] = y.v[0];
      }
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
  // Heads side by side where they are closer together than tokens and leave a
  // warp at least as many steps as it has copies under way; with fewer it
  // mostly starts and ends (4 x 8192 tokens of 16 + 4 heads of 64, 2.5 steps:
  // 35.5 us, 31.2 with tokens side by side; of 32 + 8 heads, 5 steps: 30.2, 31.4).
  p.over_heads = near[2] <= near[1] && p.heads >= kDepth * groups ? 1 : 0;
  const long long tokens = a.batch * a.length;
  const long long rows = p.over_heads ? tokens : (tokens + groups - 1) / groups;
  // The heads of a token are divided among warps so that the last wave of
  // blocks is not a small one: the division with the least waves x (steps of a
  // warp + 4), where 4 stands for what a warp does once. 2 x 8192 tokens of 16
  // + 8 heads of 128: 38.0 us undivided (1.2 waves), 35.3 in two; 2 x 4096 of
  // 8 + 8 heads of 64: 7.9 in three (0.9 waves), 8.8 in four (1.2). From
  // kManyWaves on, the last one no longer counts.
  const int hstep = p.over_heads ? groups : 1;
  const int steps = (p.heads + hstep - 1) / hstep;
  const long long slots = static_cast<long long>(kBlocksPerSm) * sm_count() * (kThreads / 32);
  long long best = 0;
  if (rows * steps <= slots) p.chunk = hstep;  // all in one wave
  for (int n = 1; rows * steps > slots && n <= std::min(steps, kMaxDivision); ++n) {
    const long long per = (steps + n - 1) / n, waves = (rows * ((steps + per - 1) / per) + slots - 1) / slots;
    if (best == 0 || waves * (per + 4) < best) {
      best = waves * (per + 4);
      p.chunk = static_cast<int>(per) * hstep;
    }
    if (waves >= kManyWaves) break;
  }
  p.n_chunks = static_cast<uint32_t>((p.heads + p.chunk - 1) / p.chunk);
  const long long warps = rows * p.n_chunks;
  if (warps > 0x7fffffff) return cudaErrorInvalidConfiguration;
  p.tokens = static_cast<uint32_t>(tokens);
  p.length = static_cast<uint32_t>(a.length);
  p.warps = static_cast<uint32_t>(warps);
  const int blocks = static_cast<int>((warps + kThreads / 32 - 1) / (kThreads / 32));
  auto kern = a.interleaved ? rotary_kernel<T, VEC, true> : rotary_kernel<T, VEC, false>;
  constexpr int smem = VEC > 1 ? 2 * kDepth * kThreads * 16 : 0;
  static std::atomic<bool> configured[2][kMaxFlagDevices];
  const cudaError_t e = ensure_smem_limit(kern, smem, configured[a.interleaved ? 1 : 0]);
  return e == cudaSuccess ? launch_pdl(kern, blocks, kThreads, smem, stream, p) : e;
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
  if (a.slots != nullptr && (a.page_size <= 0 || a.cache_blocks < 0))
    return fail(FL_ERR_INVALID_ARGUMENT, "page_size must be positive");
  if ((a.heads > 0 && (!a.q || !a.q_out)) || (a.kv_heads > 0 && (!a.k || !a.k_out)) || (!a.table && a.rot > 0))
    return fail(FL_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if ((a.slots != nullptr) != (a.v != nullptr) || (a.v != nullptr && !a.v_out))
    return fail(FL_ERR_INVALID_ARGUMENT, "the cache form takes v, its cache and the slots together");
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
