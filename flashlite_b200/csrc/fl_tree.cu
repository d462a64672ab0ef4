// Attention of new tokens (one, a chunk, or a tree of drafted ones) over a
// paged cache, on the tensor cores.
//
//   o_t = sum_j w_tj v_j / l_t,  w_tj = 2^(scale log2(e) q_t.k_j - m_t),
//   l_t = sum_j w_tj, over the keys j that token t sees: the cached ones and
//   the new ones that its mask (or the causal rule) names. m_t is a running
//   reference maximum; a row that sees nothing gives 0 and -inf.
//
// fl_tree_common.cuh has the units of work and their division. This file has
// the entry point and the kernel: units of up to 128 rows, S = Q K^T and
// O += P V as 128-row products, keys and values gathered page by page with
// TMA. (Units of few rows take the transposed products of fl_tree_few.cu.)
//
// A CTA is a scheduler warp, K and V producer warps, an MMA warp and one
// softmax warpgroup, one thread per row; two CTAs share an SM and fill each
// other's waits. S and O accumulate in TMEM, P goes to TMEM as operand A.
//
// Bound by the products and the softmax of a tile, and by memory only with
// few rows. 64 keys at head dimension 128, in cycles of one CTA: S 530 (its
// multiplications 256: every instruction reads its 128 rows of Q from shared
// memory again, 67 cycles for 64 keys and 79 for 128), P V 400, softmax 1,550
// with both CTAs' warps at work. 4 requests of 509 tokens x 4 heads to a key
// head over up to 8192 keys, bf16: 258 to 283 us, 720 to 790 TFLOP/s, at some
// 1.4 GHz under the power limit; 16 trees of 61 nodes x 4 heads over up to
// 5000 keys: 76 to 94 us, with 6 us to the first tile. Half of Q kept in TMEM
// took 9 % off a tile's cycles and nothing off the time. Two row tiles in one
// CTA per SM, with K and V read once for both, were slower: TMEM then holds S
// of 128 keys only with P in its place, which puts S, softmax and P V in a
// chain (273 us for 245), with 64 keys S stays as costly (336 us), and no
// second CTA fills a change of units (13,000 cycles).
//
// Keys that no row may see are kept out of the products as zeros: masked
// scores are replaced, not added to, and V rows past the visible keys are
// cleared in shared memory, since 0 times what an unused row holds may be
// NaN. Rows of V that some rows see and others do not are searched for
// infinities and NaN, which are cleared too and added back, in the epilogue,
// to the rows that see them.
//
// P is rounded to the 16-bit type of V, since both operands of a tensor
// instruction have one type: a probability is off by 2^-11 (fp16) or 2^-8
// (bf16) of itself, and a result by that much of sum_j p_j |v_j| at most.
// Against 64 bits the results are 1.2 to 1.4 times as far off as those of a
// 32-bit computation that rounds its output alone (trees in fp16 2.9e-4 for
// 2.1e-4 of the norm, decoding in bf16 2.3e-3 for 1.7e-3). Scores, statistics,
// sums, O and parts are fp32.

#include <algorithm>
#include <cmath>
#include <string>

#include "fl_tree_common.cuh"

namespace fl {
namespace {

constexpr int kThreads = 256;
constexpr int kBM = 128;           // rows per unit (UMMA M)
constexpr int kMaxRequests = 4096;
constexpr uint32_t kTmemCols = 256;
constexpr int kSegReaders = 7;     // K, V, MMA and four softmax warps
constexpr int kCtasPerSm = 2;
// Units of more rows look before they write a part whether they are the last
// (tree of 61 nodes x 4 heads: 99 -> 89 us); with few rows the look costs more
// than the part (3 us on the smallest calls).
constexpr int kDirectRows = 32;
// What a change of units costs in tiles: of 0, 2, 3, 4, 6, 8 and 12, 3 is best
// or within 2 % of it (40 requests x 8 tokens over 6000 keys 105 us for 110,
// 4 prompts of 1000 38 for 42, chunks 258 for 270).
constexpr int kGapTiles = 3;

// Shape per head dimension; tiles are made of 64-column (128-byte) swizzle
// atoms as in the other forward kernels. K and V tiles are 16 KB both ways;
// two CTAs share an SM's 228 KB.
//   TMEM columns: S (kBN) | O (HD) | P (kBN / 2): 256 and 224.
template <int HD>
struct Shape {
  static_assert(HD == 64 || HD == 128, "head dimension 64 or 128");
  static constexpr int kBN = HD == 64 ? 128 : 64;
  static constexpr int kHalves = HD / 64;
  static constexpr int kStagesK = 3;
  static constexpr int kStagesV = HD == 64 ? 3 : 2;
  static constexpr int kQBytes = kBM * HD * 2;
  static constexpr int kTileBytes = kBN * HD * 2;
  static constexpr int kSmemQ = 0;
  static constexpr int kSmemK = kSmemQ + kQBytes;
  static constexpr int kSmemV = kSmemK + kStagesK * kTileBytes;
  static constexpr int kSmemMisc = kSmemV + kStagesV * kTileBytes;
  static constexpr int kSmemBytes = kSmemMisc + 1024;
  static constexpr uint32_t kColS = 0, kColO = kBN, kColP = kBN + HD;
  static_assert(kColP + kBN / 2 <= kTmemCols, "TMEM");
  static_assert(2 * (kSmemBytes + 1024) <= 228 * 1024, "two CTAs per SM");
};
// Register split between the producer, MMA and scheduler warps and the softmax
// warps, whose row of scores is 128 registers at head dimension 64 and 64 at
// 128: 128 * (72 + 184) = 128 * (88 + 168) = 256 * 128, the launch's total.
// (At 128, 64 + 192 spilled in the MMA warp: tree 98 us for 87, chunk 303 for
// 282. At 64 the compiler spills 64 bytes a thread with the split taken.)
template <int HD>
constexpr int kRegsProducer = HD == 64 ? 72 : 88;
template <int HD>
constexpr int kRegsSoftmax = 256 - kRegsProducer<HD>;

// Joins the n partial results base, base + stride, ... of a unit:
//   o = sum_k l_k 2^(m_k - M) o_k / sum_k l_k 2^(m_k - M),  M = max_k m_k,
// by the 128 softmax threads; into slot `to` or, if to < 0, out. Part i of a
// unit that begins in CTA `first` is slot 2 first + 1 (i = 0) or 2 (first + i).
// Neighbouring threads take neighbouring rows (the layout of a slot is
// [D / 4][128] float4), and the columns that few rows leave threads for.
// Returns the joined reference and sum of row tid, if tid < rows.
template <typename T, int HD>
__device__ __forceinline__ float2 join_parts(const TreeParams& p, const Segment& g, int tid, int first, int base, int stride,
                                            int n, int to) {
  constexpr int kVecs = HD / 4;
  int span = 1;  // rows, as a power of two
  while (span < g.rows) span *= 2;
  const int row = tid & (span - 1), lanes = kBM / span, c0 = tid / span;
  if (row >= g.rows || c0 >= kVecs) return make_float2(0.0f, 0.0f);
  const int token = g.begin + g.i0 + row / p.group, head = g.head * p.group + row % p.group;
  const long long orow = static_cast<long long>(token) * p.heads + head;
  float2 joined = make_float2(-INFINITY, 0.0f);
  // kCols columns (of four) of kBatch parts at a time, all their loads under
  // way together. Rolled otherwise: on its first run in a kernel, code costs
  // as much to fetch as to execute.
  auto join = [&](auto cols, auto batch) {
    constexpr int kCols = decltype(cols)::value, kBatch = decltype(batch)::value;
#pragma unroll 1
    for (int c = c0; c < kVecs; c += kCols * lanes) {
      float acc[4 * kCols], m = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 4 * kCols; ++j) acc[j] = 0.0f;
#pragma unroll 1
      for (int k0 = 0; k0 < n; k0 += kBatch) {
        float2 l[kBatch];
        float v[kBatch][4 * kCols];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const bool in = k0 + k < n;
          const int sl = slot_of(first, base + min(k0 + k, n - 1) * stride);
          l[k] = in ? __ldcg(p.part_sum + sl * kBM + row) : make_float2(-INFINITY, 0.0f);
          const float4* from = reinterpret_cast<const float4*>(p.part) + static_cast<long long>(sl) * kVecs * kBM + row;
#pragma unroll
          for (int j = 0; j < kCols; ++j)
            get4(v[k] + 4 * j, in && c + j * lanes < kVecs ? __ldcg(from + (c + j * lanes) * kBM)
                                                           : make_float4(0.f, 0.f, 0.f, 0.f));
        }
        join_step<kBatch, 4 * kCols>(m, sum, acc, l, v);
      }
      const float inv = join_inv(sum);
      joined = make_float2(m, sum);
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        if (c + j * lanes >= kVecs) break;
        const float4 o = make_float4(acc[4 * j] * inv, acc[4 * j + 1] * inv, acc[4 * j + 2] * inv, acc[4 * j + 3] * inv);
        if (to >= 0)
          reinterpret_cast<float4*>(p.part)[(static_cast<long long>(to) * kVecs + c + j * lanes) * kBM + row] = o;
        else
          reinterpret_cast<uint2*>(static_cast<T*>(p.out) + orow * HD)[c + j * lanes] =
              make_uint2(pack2<T>(o.x, o.y), pack2<T>(o.z, o.w));
      }
    }
  };
  static_assert(kDirectRows >= 32, "units that are joined from registers take the first form");
  if (lanes * 4 <= kVecs) join(std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{});
  else join(std::integral_constant<int, 1>{}, std::integral_constant<int, 6>{});
  if (c0 == 0 && to < 0 && p.lse != nullptr) p.lse[orow] = join_lse(joined.x, joined.y) * 0.69314718055994531f;
  return joined;
}

template <typename T, int HD, bool kAligned>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) tree_attention_kernel(const __grid_constant__ TreeParams p) {
  using C = Shape<HD>;
  constexpr int kBN = C::kBN;
  constexpr int kStagesK = C::kStagesK, kStagesV = C::kStagesV;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  const uint32_t s_q = sbase + C::kSmemQ, s_k0 = sbase + C::kSmemK, s_v0 = sbase + C::kSmemV;
  // misc block: barriers | segments | flags
  const uint32_t bars = sbase + C::kSmemMisc;
  const uint32_t bar_kfull = bars, bar_kempty = bar_kfull + 8 * kStagesK;
  const uint32_t bar_vfull = bar_kempty + 8 * kStagesK, bar_vempty = bar_vfull + 8 * kStagesV;
  const uint32_t bar_segfull = bar_vempty + 8 * kStagesV, bar_segempty = bar_segfull + 8 * kSegRing;
  const uint32_t bar_x = bar_segempty + 8 * kSegRing;
  const uint32_t bar_qfull = bar_x, bar_qfree = bar_x + 8, bar_s = bar_x + 16, bar_sfree = bar_x + 24, bar_p = bar_x + 32,
                 bar_pv = bar_x + 40, bar_ofree = bar_x + 48, bar_seg = bar_x + 56, bar_drain = bar_x + 64,
                 bar_join = bar_x + 72;
  const uint32_t bar_count = bar_x + 80;  // arrival counts ready: one for each of the CTA's (up to) two parts
  constexpr int kBarBytes = 8 * (2 * kStagesK + 2 * kStagesV + 2 * kSegRing + 12);
  constexpr int kSegOff = (kBarBytes + 15) / 16 * 16;
  uint8_t* misc = smem + C::kSmemMisc;
  Segment* segs = reinterpret_cast<Segment*>(misc + kSegOff);
  constexpr int kFlagOff = kSegOff + kSegRing * static_cast<int>(sizeof(Segment));
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc + kFlagOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + kFlagOff + 4);
  volatile int* bad_flag = reinterpret_cast<volatile int*>(misc + kFlagOff + 8);
  volatile int* last_flag = reinterpret_cast<volatile int*>(misc + kFlagOff + 12);
  // One word for each of the CTA's (up to) two parts: the first softmax warp can
  // be at the second part's decision while another has yet to read the first
  // part's, which a meeting's end does not hold it back from.
  volatile int* direct_flag = reinterpret_cast<volatile int*>(misc + kFlagOff + 16);
  static_assert(kFlagOff + 24 <= 1024, "misc block");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x;

  // ---- setup ----
  if (tid == 0) {
    for (int st = 0; st < kStagesK; ++st) {
      mbar_init(bar_kfull + 8 * st, 1);
      mbar_init(bar_kempty + 8 * st, 1);
    }
    for (int st = 0; st < kStagesV; ++st) {
      mbar_init(bar_vfull + 8 * st, 1);
      mbar_init(bar_vempty + 8 * st, 1);
    }
    for (int st = 0; st < kSegRing; ++st) {
      mbar_init(bar_segfull + 8 * st, 1);
      mbar_init(bar_segempty + 8 * st, kSegReaders);
    }
    mbar_init(bar_qfull, 1);
    mbar_init(bar_qfree, 1);
    mbar_init(bar_count, 1);
    mbar_init(bar_count + 8, 1);
    mbar_init(bar_join, 4);
    mbar_init(bar_s, 1);
    mbar_init(bar_sfree, 4);  // one arrival per softmax warp
    mbar_init(bar_p, 4);
    mbar_init(bar_pv, 1);
    mbar_init(bar_ofree, 4);
    mbar_init(bar_seg, 1);
    mbar_init(bar_drain, 1);
    *abort_flag = 0;
    *bad_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.tm_q);
    tma_prefetch_desc(&p.tm_k);
    tma_prefetch_desc(&p.tm_v);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), kTmemCols);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kRegsProducer<HD>));
    if (warp == 3) {
      // ======================= scheduler =======================
      Scheduler<kBN, kAligned, kGapTiles> sched(p, cta, lane);
      for (int ring = 0;; ++ring) {
        const Segment g = sched.next();
        const int st = ring % kSegRing;
        if (!wait_all(bar_segempty + 8 * st, ((ring / kSegRing) & 1) ^ 1, abort_flag, p.err)) break;
        if (lane == 0) {
          segs[st] = g;
          mbar_arrive(bar_segfull + 8 * st);
        }
        __syncwarp();
        if (g.t1 < 0) break;
        if (g.slot >= 0) {
          ready_counts(p, g, cta, lane, join_group(g));
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_count + 8 * (g.slot & 1));
        }
      }
      clear_padding<T, HD>(p, cta, p.grid, lane);
    } else if (warp == 0 || warp == 2) {
      // ======================= K (and Q) producer, V producer =======================
      const bool is_k = warp == 0;
      const int stages = is_k ? kStagesK : kStagesV;
      const CUtensorMap* tm = is_k ? &p.tm_k : &p.tm_v;
      const uint32_t ring0 = is_k ? s_k0 : s_v0, full0 = is_k ? bar_kfull : bar_vfull, empty0 = is_k ? bar_kempty : bar_vempty;
      int tile = 0, seg = 0, q_loads = 0;
      bool ok = true;
      while (ok) {
        const int sl = seg % kSegRing;
        if (!wait_all(bar_segfull + 8 * sl, (seg / kSegRing) & 1, abort_flag, p.err)) break;
        const Segment g = segs[sl];
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_segempty + 8 * sl);
        ++seg;
        if (g.t1 < 0) break;
        PageNumbers<kBN> pages(p, g, lane);
        if (is_k) {
          if (!wait_all(bar_qfree, ((seg - 1) & 1) ^ 1, abort_flag, p.err)) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(bar_qfull, p.group * p.tile_tokens * 128 * C::kHalves);
#pragma unroll
            for (int hh = 0; hh < C::kHalves; ++hh)
              tma_load_3d(s_q + hh * (kBM * 128), &p.tm_q, bar_qfull, 64 * hh, g.head * p.group, g.begin + g.i0);
          }
          __syncwarp();
          ++q_loads;
        }
        for (int t = g.t0; t < g.t1; ++t, ++tile) {
          pages.begin_tile(t);
          const int st = tile % stages;
          if (!wait_all(empty0 + 8 * st, ((tile / stages) & 1) ^ 1, abort_flag, p.err)) {
            ok = false;
            break;
          }
          load_tile<HD, kBN>(p, tm, pages, g, t, ring0 + st * C::kTileBytes, full0 + 8 * st, 0, 1, is_k);
        }
      }
      if (*abort_flag && lane == 0) {
        // let every copy this warp started land before shared memory is released
        for (int t = tile > stages ? tile - stages : 0; t < tile; ++t)
          mbar_wait_quiet(full0 + 8 * (t % stages), (t / stages) & 1);
        if (q_loads > 0) mbar_wait_quiet(bar_qfull, (q_loads - 1) & 1);
      }
    } else {
      // ======================= MMA issuer =======================
      constexpr uint32_t idesc_s = make_idesc_f16_f32(kBM, kBN, false, false, kBf16);
      constexpr uint32_t idesc_pv = make_idesc_f16_f32(kBM, HD, true, false, kBf16);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint64_t dq = make_sdesc_sw128(s_q, 16, 1024);
      const uint64_t dk0 = make_sdesc_sw128(s_k0, 16, 1024);
      const uint64_t dv0 = make_sdesc_sw128(s_v0, HD == 64 ? 8192 : kBN * 128, 1024);
      constexpr uint64_t kStageEnc = C::kTileBytes >> 4, kQHalf = (kBM * 128) >> 4, kKHalf = (kBN * 128) >> 4;
      auto ready = [&](uint32_t bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, mbar_try_wait_hint(bar, parity, FL_ISSUER_HINT_NS));
      };
      // Keeps trying until the step is done; bounded like every wait.
      auto until = [&](auto&& step) -> bool {
        if (step()) return true;
        const uint64_t t0 = globaltimer_ns();
        while (true) {
#pragma unroll 1
          for (int k = 0; k < 64; ++k)
            if (step()) return true;
          const bool late = globaltimer_ns() - t0 > FL_WAIT_LIMIT_NS;
          if (__any_sync(0xffffffffu, late || *abort_flag)) {
            if (lane == 0 && !*abort_flag) {
              *abort_flag = 1;
              if (p.err) atomicOr(p.err, kDevErrWaitTimeout);
            }
            return false;
          }
        }
      };
      int ks = 0, vs = 0, seg = 0;  // S products, P V products, segments so far
      bool ok = true;
      while (ok) {
        const int sl = seg % kSegRing;
        if (!wait_all_issuer(bar_segfull + 8 * sl, (seg / kSegRing) & 1, abort_flag, p.err)) break;
        const Segment g = segs[sl];
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_segempty + 8 * sl);
        if (g.t1 < 0) break;
        if (!wait_all_issuer(bar_qfull, seg & 1, abort_flag, p.err)) break;
        auto try_s = [&](bool last) -> bool {
          const int st = ks % kStagesK;
          if (!ready(bar_kfull + 8 * st, (ks / kStagesK) & 1) || !ready(bar_sfree, (ks & 1) ^ 1)) return false;
          tc_fence_after();
          const uint64_t bd = dk0 + st * kStageEnc;
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
              umma_f16_ss(tm + C::kColS, dq + 2 * (kk & 3) + (kk >> 2) * kQHalf, bd + 2 * (kk & 3) + (kk >> 2) * kKHalf,
                          idesc_s, kk > 0 ? 1u : 0u);
            umma_commit(bar_s);
            umma_commit(bar_kempty + 8 * st);
            if (last) umma_commit(bar_qfree);
          }
          __syncwarp();
          ++ks;
          return true;
        };
        ok = until([&] { return try_s(g.t0 + 1 == g.t1); });
        // O of the segment before has been read
        if (ok) ok = wait_all_issuer(bar_ofree, (seg & 1) ^ 1, abort_flag, p.err);
        if (!ok) break;
        if (lane == 0) *bad_flag = 0;
        // keys from here on are hidden from some row of the tile
        const int mixed = p.mask != nullptr ? g.ctx : min(g.ctx + g.i0 + 1, g.keys);
        uint32_t accumulate = 0;
        for (int t = g.t0; ok && t < g.t1; ++t) {
          // The next S and this tile's P V, in the order in which they can go:
          // a V tile is not held while the next K tile is awaited.
          const int st = vs % kStagesV;
          bool s_done = t + 1 == g.t1, pv_done = false, guarded = false;
          auto try_pv = [&]() -> bool {
            if (!guarded) {
              if (!ready(bar_vfull + 8 * st, (vs / kStagesV) & 1)) return false;
              const int valid = min(kBN, g.keys - t * kBN), from = max(0, min(mixed - t * kBN, valid));
              if (from < kBN) {
                const bool bad = guard_v<T, HD, kBN>(s_v0 + st * C::kTileBytes, from, valid, lane);
                if (bad && lane == 0) *bad_flag = 1;
                __syncwarp();
              }
              guarded = true;
            }
            if (!ready(bar_p, vs & 1)) return false;
            tc_fence_after();
            const uint64_t bd = dv0 + st * kStageEnc;
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < kBN / 16; ++kk)
                umma_f16_ts(tm + C::kColO, tm + C::kColP + kk * 8, bd + 128 * kk, idesc_pv, kk > 0 ? 1u : accumulate);
              umma_commit(bar_pv);
              umma_commit(bar_vempty + 8 * st);
            }
            __syncwarp();
            return true;
          };
          ok = until([&]() -> bool {
            if (!s_done) s_done = try_s(t + 2 == g.t1);
            if (!pv_done) pv_done = try_pv();
            return s_done && pv_done;
          });
          accumulate = 1;
          ++vs;
        }
        if (lane == 0) mbar_arrive(bar_seg);  // publishes bad_flag
        __syncwarp();
        ++seg;
      }
      // wait until every MMA this warp issued has completed
      if (elect_one()) {
        umma_commit(bar_drain);
        mbar_wait_quiet(bar_drain, 0);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kRegsSoftmax<HD>));
    // ======================= softmax: one thread per row =======================
    const int t_row = tid - 128;
    const uint32_t lane_base = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t tS = tmem + lane_base + C::kColS, tP = tmem + lane_base + C::kColP, tO = tmem + lane_base + C::kColO;
    const int my_token = t_row / p.group, my_head = t_row % p.group;  // within the row tile
    const float sc = p.scale_log2;
    const bool prescale = !(sc > 0.0f);  // a negative scale turns maxima into minima: applied first
    int js = 0, seg = 0, joins = 0;      // tiles, segments and meetings so far
    bool ok = true;
    // the four warps meet with bounded waits: one that has given up does not come
    auto meet = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_join);
      return wait_all(bar_join, joins++ & 1, abort_flag, p.err);
    };
    while (ok) {
      const int sl = seg % kSegRing;
      if (!wait_all(bar_segfull + 8 * sl, (seg / kSegRing) & 1, abort_flag, p.err)) break;
      const Segment g = segs[sl];
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_segempty + 8 * sl);
      if (g.t1 < 0) break;
      const bool live_warp = 32 * (warp & 3) < g.rows;  // warps without rows only keep the barriers going
      const bool live = t_row < g.rows;
      const int token = g.begin + g.i0 + my_token;      // row of q, if live
      // keys this row sees without looking at its mask, and where its mask ends
      const int plain = p.mask != nullptr ? min(g.ctx, g.keys) : min(g.ctx + g.i0 + my_token + 1, g.keys);
      const uint32_t* words = p.mask != nullptr && live ? p.mask + static_cast<long long>(token) * p.mask_words : nullptr;
      float m_ref = -INFINITY, l = 0.0f, l_fix = 0.0f;
      for (int t = g.t0; t < g.t1; ++t, ++js) {
        if (!(ok = wait_all(bar_s, js & 1, abort_flag, p.err))) break;
        if (!live_warp) {
          if (lane == 0) mbar_arrive(bar_sfree);
          if (t > g.t0 && !(ok = wait_all(bar_pv, (js - 1) & 1, abort_flag, p.err))) break;
          if (lane == 0) mbar_arrive(bar_p);
          continue;
        }
        tc_fence_after();
        uint32_t sr[kBN];
        if constexpr (kBN == 128) tmem_ld128_wait(tS, sr);
        else tmem_ld64_wait(tS, sr);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_sfree);
        float s[kBN];
#pragma unroll
        for (int c = 0; c < kBN; ++c) s[c] = __uint_as_float(sr[c]);
        float scl = sc;
        if (prescale) {
#pragma unroll
          for (int c = 0; c < kBN; ++c) s[c] *= sc;
          scl = 1.0f;
        }
        const int k0 = t * kBN;
        if (__any_sync(0xffffffffu, plain < k0 + kBN)) {
#pragma unroll
          for (int q = 0; q < kBN / 32; ++q) {
            // bit c: column 32 q + c is visible
            const int first = plain - (k0 + 32 * q);
            uint32_t vis = first <= 0 ? 0u : first >= 32 ? 0xffffffffu : (1u << first) - 1u;
            if (words != nullptr && first < 32) {
              const int j0 = k0 + 32 * q - g.ctx;  // new token of column 0; may be negative
              const int w = j0 >> 5, sh = j0 & 31;
              const uint32_t lo = w >= 0 && w < p.mask_words ? words[w] : 0u;
              const uint32_t hi = w + 1 >= 0 && w + 1 < p.mask_words ? words[w + 1] : 0u;
              uint32_t bits = __funnelshift_r(lo, hi, sh);
              const int end = g.keys - (k0 + 32 * q);
              if (end < 32) bits &= end <= 0 ? 0u : (1u << end) - 1u;
              vis |= bits;
            }
#pragma unroll
            for (int c = 0; c < 32; ++c) s[32 * q + c] = (vis >> c & 1u) ? s[32 * q + c] : -INFINITY;
          }
        }
        float mx;
        {
          float part[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            constexpr int L = kBN / 4;
            float a = fmaxf(s[q * L], s[q * L + 1]);
#pragma unroll
            for (int e = 2; e < L; e += 2) a = fmax3(a, s[q * L + e], s[q * L + e + 1]);
            part[q] = a;
          }
          mx = fmax3(fmaxf(part[0], part[1]), part[2], part[3]);
        }
        // The argument of 2^x is one fused multiply-add, exact up to its own
        // rounding, while the reference is a rounded product: past 2^20 that
        // rounding alone could empty a row, and scores are scaled first.
        const float mag = fabsf(mx * scl);
        if (__any_sync(0xffffffffu, mag > 1048576.0f && mag < INFINITY) && !prescale) {
#pragma unroll
          for (int c = 0; c < kBN; ++c) s[c] *= sc;
          mx *= sc;
          scl = 1.0f;
        }
        const float m_new = fmaxf(m_ref, mx * scl);
        const bool need = m_new > m_ref + kLag;
        float alpha = 1.0f;
        if (need) {
          alpha = ex2_approx(m_ref - m_new);
          m_ref = m_new;
        }
        l *= alpha;
        l_fix *= alpha;
        const float m_use = (m_ref == -INFINITY) ? 0.0f : m_ref - kUp;
        const float2 scl2 = make_float2(scl, scl), nm2 = make_float2(-m_use, -m_use);
        float2 sum[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t pk[kBN / 2];
#pragma unroll
        for (int e = 0; e < kBN / 2; ++e) {
          const float2 x = __ffma2_rn(make_float2(s[2 * e], s[2 * e + 1]), scl2, nm2);
          const float2 pp = make_float2(ex2_approx(x.x), ex2_approx(x.y));
          sum[e & 3] = __fadd2_rn(sum[e & 3], pp);
          pk[e] = pack2<T>(pp.x, pp.y);
        }
        {
          const float2 a = __fadd2_rn(sum[0], sum[1]), b = __fadd2_rn(sum[2], sum[3]);
          l += (a.x + a.y) + (b.x + b.y);
          // The tile's largest p enters O rounded: O's normaliser sees the
          // same value, so that a row which one key dominates gives that
          // key's value exactly; the log-sum-exp keeps the unrounded sum.
          const float pm = ex2_approx(fmaf(mx, scl, -m_use));
          l_fix += static_cast<float>(static_cast<T>(pm)) - pm;
        }
        // P V of the tile before: its P is free to be overwritten, O to be rescaled
        if (t > g.t0) {
          if (!(ok = wait_all(bar_pv, (js - 1) & 1, abort_flag, p.err))) break;
          tc_fence_after();
          if (__any_sync(0xffffffffu, need)) {
            uint32_t o[32];
#pragma unroll
            for (int h = 0; h < HD / 32; ++h) {
              tmem_ld32_wait(tO + h * 32, o);
#pragma unroll
              for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
              tmem_st32(tO + h * 32, o);
            }
          }
        }
#pragma unroll
        for (int q = 0; q < kBN / 32; ++q)
          tmem_st16(tP + q * 16, *reinterpret_cast<const uint32_t(*)[16]>(&pk[q * 16]));
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p);
      }
      if (!ok) break;

      // A part whose unit's other parts are all there already is joined from
      // its registers and never written: as a rule a unit's later part ends
      // while the CTA of its first part is still at work.
      const int first = cta - g.part;
      bool direct = false;
      if (g.slot >= 0 && g.parts <= kJoinMany && g.rows > kDirectRows) {
        if (t_row == 0)
          direct_flag[g.slot & 1] = mbar_wait(bar_count + 8 * (g.slot & 1), 0, abort_flag, p.err) &&
                                    others_arrived(group_word(p, g, cta, kJoinMany), p.tag, g.parts);
        if (!(ok = meet())) break;
        direct = direct_flag[g.slot & 1] != 0;
      }

      // ---- epilogue of the segment ----
      if (!(ok = wait_all(bar_pv, (js - 1) & 1, abort_flag, p.err))) break;
      if (!(ok = wait_all(bar_seg, seg & 1, abort_flag, p.err))) break;
      tc_fence_after();
      if (live_warp) {
        const bool bad = *bad_flag != 0;
        const float norm = l + l_fix;
        const float inv = (l > 0.0f) ? 1.0f / norm : 0.0f;
        const float lse2 = (l == 0.0f) ? -INFINITY : (m_ref - kUp) + log2f(l);
        const long long orow = static_cast<long long>(token) * p.heads + g.head * p.group + my_head;
        float4* prow = g.slot < 0 || direct
                           ? nullptr
                           : reinterpret_cast<float4*>(p.part) + static_cast<long long>(g.slot) * (HD / 4) * kBM + t_row;
        if (live) {
          if (prow != nullptr) p.part_sum[g.slot * kBM + t_row] = make_float2(m_ref - kUp, l);
          else if (!direct && p.lse != nullptr) p.lse[orow] = lse2 * 0.69314718055994531f;
        }
#pragma unroll 1
        for (int h = 0; h < HD / 32; ++h) {
          uint32_t r[32];
          __syncwarp();
          tmem_ld32_wait(tO + h * 32, r);
          float o[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = __uint_as_float(r[c]) * inv;
          if (bad && live) {
            // infinities and NaN that guard_v cleared, for the rows that see them
            const int hidden = p.mask != nullptr ? g.ctx : g.ctx + g.i0 + 1;
            for (int key = max(hidden, g.t0 * kBN); key < min(g.t1 * kBN, g.keys); ++key) {
              const int j = key - g.ctx;
              const bool seen = words != nullptr ? (j >> 5) < p.mask_words && (words[j >> 5] >> (j & 31) & 1u)
                                                 : key < plain;
              if (!seen) continue;
              const int blk = p.table[g.request * p.table_stride + (key >> p.page_shift)];
              if (blk < 0 || blk >= p.num_blocks) continue;
              const T* vr = static_cast<const T*>(p.v) + blk * p.v_stride[0] +
                            (key & ((1 << p.page_shift) - 1)) * p.v_stride[1] + g.head * p.v_stride[2] + 32 * h;
#pragma unroll
              for (int c = 0; c < 32; ++c) {
                const float x = static_cast<float>(vr[c]);
                if (!(fabsf(x) < INFINITY)) o[c] += x;
              }
            }
          }
          if (direct && live) {
            // as join_parts does it, with this part from its registers
            float acc[32], m = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int c = 0; c < 32; ++c) acc[c] = 0.0f;
#pragma unroll 1
            for (int k0 = 0; k0 < g.parts; k0 += 2) {
              float2 l2[2];
              float v[2][32];
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const bool in = k0 + k < g.parts, mine = k0 + k == g.part;
                const int sl = slot_of(first, min(k0 + k, g.parts - 1));
                l2[k] = !in    ? make_float2(-INFINITY, 0.0f)
                        : mine ? make_float2(m_ref - kUp, l)
                               : __ldcg(p.part_sum + sl * kBM + t_row);
                const float4* from = reinterpret_cast<const float4*>(p.part) +
                                     (static_cast<long long>(sl) * (HD / 4) + 8 * h) * kBM + t_row;
#pragma unroll
                for (int c = 0; c < 8; ++c)
                  get4(v[k] + 4 * c, in && !mine ? __ldcg(from + c * kBM) : make_float4(0.f, 0.f, 0.f, 0.f));
#pragma unroll
                for (int c = 0; c < 32; ++c) v[k][c] = mine ? o[c] : v[k][c];
              }
              join_step<2, 32>(m, sum, acc, l2, v);
            }
            const float joined = join_inv(sum);
#pragma unroll
            for (int c = 0; c < 32; ++c) o[c] = acc[c] * joined;
            if (h == 0 && p.lse != nullptr) p.lse[orow] = join_lse(m, sum) * 0.69314718055994531f;
          }
          if (live) {
            if (prow != nullptr) {
#pragma unroll
              for (int c = 0; c < 32; c += 4)
                prow[(8 * h + c / 4) * kBM] = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
            } else {
              uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + orow * HD + 32 * h);
#pragma unroll
              for (int c = 0; c < 4; ++c)
                to[c] = make_uint4(pack2<T>(o[8 * c], o[8 * c + 1]), pack2<T>(o[8 * c + 2], o[8 * c + 3]),
                                   pack2<T>(o[8 * c + 4], o[8 * c + 5]), pack2<T>(o[8 * c + 6], o[8 * c + 7]));
            }
          }
        }
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_ofree);
      ++seg;
      if (g.slot >= 0 && !direct) {
        // a part: whoever arrives last joins, within its group of parts and then among the groups
        const int size = join_group(g), groups = g.parts <= size ? 1 : (g.parts + size - 1) / size;
        int base = group_base(g, size), stride = 1, n = min(size, g.parts - base);
#pragma unroll 1
        while (true) {
          if (!(ok = meet())) break;  // all of this CTA's part is written
          if (t_row == 0)
            *last_flag = mbar_wait(bar_count + 8 * (g.slot & 1), 0, abort_flag, p.err) &&
                         arrive_last(stride == 1 ? group_word(p, g, cta, size) : unit_word(p, g, cta), n);
          if (!(ok = meet())) break;
          if (*last_flag == 0) break;
          const int to = stride == 1 && groups > 1 ? slot_of(first, base) : -1;
          const float2 joined = join_parts<T, HD>(p, g, t_row, first, base, stride, n, to);
          if (to < 0) break;
          if (!(ok = meet())) break;  // the group's sums have been read: its first slot takes the joined ones
          if (live) p.part_sum[to * kBM + t_row] = joined;
          base = 0;
          stride = size;
          n = groups;
        }
      }
    }
  }

  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
size_t workspace_bytes(int grid, int64_t head_dim) {
  const size_t slots = 2 * static_cast<size_t>(grid);
  return slots * kBM * (head_dim + 2) * sizeof(float) + 3 * grid * sizeof(unsigned long long);
}

bool encode(CUtensorMap* tm, bool bf16, const void* base, int rank, const cuuint64_t* dims, const int64_t* strides,
            const cuuint32_t* box) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return false;
  cuuint64_t bytes[3];
  cuuint32_t one[4] = {1, 1, 1, 1};
  // the stride of a dimension of size 1 is never used, and torch gives it any value
  for (int i = 0; i + 1 < rank; ++i) bytes[i] = dims[i + 1] == 1 ? dims[0] * 2 : static_cast<cuuint64_t>(strides[i]) * 2;
  return enc(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(base),
             dims, bytes, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD, bool kAligned>
cudaError_t launch_kernel(const TreeParams& p, cudaStream_t stream) {
  auto kern = tree_attention_kernel<T, HD, kAligned>;
  static std::atomic<bool> configured[kMaxFlagDevices];
  const cudaError_t e = ensure_smem_limit(kern, Shape<HD>::kSmemBytes, configured);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, p.grid, kThreads, Shape<HD>::kSmemBytes, stream, p);
}

template <typename T, int HD>
cudaError_t launch(TreeParams& p, const fl_tree_attention_args& a, int64_t rows, cudaStream_t stream) {
  p.grid = kCtasPerSm * sm_count();
  p.tile_tokens = kBM / p.group;
  p.part_sum = reinterpret_cast<float2*>(p.part + 2LL * p.grid * kBM * HD);
  p.arrived = reinterpret_cast<unsigned long long*>(p.part_sum + 2LL * p.grid * kBM);
  if (!encode_tree_maps(p, a, Shape<HD>::kBN)) return cudaErrorInvalidValue;
  // The aligned division pays where units are few (16 requests x 8 tokens x 2
  // key heads over 2000 keys, head dimension 128: 17.6 us for 22.1); elsewhere
  // its code costs 2 % and it would not be taken.
  const int64_t units = a.requests * p.kv_heads * std::max<int64_t>(1, (rows + kBM - 1) / kBM);
  return 2 * units <= p.grid ? launch_kernel<T, HD, true>(p, stream) : launch_kernel<T, HD, false>(p, stream);
}

// A tag that no earlier call of this process had (the counter goes through
// 48 bits before it repeats), spread so that what other data leave in the
// workspace is unlikely to look like one.
unsigned long long next_tag() {
  static std::atomic<unsigned long long> calls{0};
  return ((calls.fetch_add(1, std::memory_order_relaxed) + 1) * 0x9E3779B97F4A7C15ull) & 0xffffffffffffull;
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
  if (a.kv_heads == 0 ? a.heads != 0 : (a.heads % a.kv_heads != 0 || a.heads / a.kv_heads > kBM))
    return fail(FL_ERR_INVALID_ARGUMENT, "heads must be a multiple of kv_heads, at most 128 times");
  if (a.page_size < 8 || a.page_size > 256 || (a.page_size & (a.page_size - 1)) != 0)
    return fail(FL_ERR_UNSUPPORTED, "page_size must be a power of two from 8 to 256");
  if (a.requests > kMaxRequests) return fail(FL_ERR_UNSUPPORTED, "at most 4096 requests");
  if (a.tokens > (1LL << 28) || a.heads > (1LL << 15) || a.num_blocks >= 0x7fffffffLL || a.table_cols > (1LL << 26) ||
      a.mask_words > (1LL << 20))
    return fail(FL_ERR_INVALID_ARGUMENT, "dimension too large");
  if (a.tokens == 0 || a.heads == 0) return FL_OK;
  if (!a.q || !a.out || !a.cu_seqlens || (a.requests > 0 && !a.context_lens) ||
      (a.requests > 0 && a.table_cols > 0 && !a.block_table) || (a.num_blocks > 0 && (!a.k_cache || !a.v_cache)))
    return fail(FL_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (a.num_blocks == 0) return fail(FL_ERR_INVALID_ARGUMENT, "empty cache");
  if (!aligned16(a.q) || !aligned16(a.k_cache) || !aligned16(a.v_cache) || !aligned16(a.out) || !aligned16(a.workspace))
    return fail(FL_ERR_MISALIGNED, "q, the caches, out and workspace must be 16-byte aligned");
  const int64_t sizes[8] = {a.tokens, a.heads, a.num_blocks, a.page_size, a.kv_heads, a.num_blocks, a.page_size, a.kv_heads};
  const int64_t strides[8] = {a.q_stride[0], a.q_stride[1], a.k_stride[0], a.k_stride[1], a.k_stride[2],
                              a.v_stride[0], a.v_stride[1], a.v_stride[2]};
  for (int i = 0; i < 8; ++i)
    if (sizes[i] > 1 && (strides[i] <= 0 || strides[i] % 8 != 0 || strides[i] >= (1LL << 39)))
      return fail(FL_ERR_MISALIGNED, "strides of q and the caches must be positive multiples of 8 elements");
  int st = check_device();
  if (st != FL_OK) return st;
  TreeParams p = {};
  if (!a.workspace || a.workspace_bytes < workspace_bytes(kCtasPerSm * sm_count(), a.head_dim))
    return fail(FL_ERR_INVALID_ARGUMENT, "workspace too small (fl_tree_attention_workspace_size)");
  p.v = a.v_cache;
  p.out = a.out;
  p.lse = a.lse;
  p.table = a.block_table;
  p.context = a.context_lens;
  p.cu = a.cu_seqlens;
  p.mask = a.tree_mask != nullptr && a.mask_words > 0 ? a.tree_mask : nullptr;
  p.part = static_cast<float*>(a.workspace);
  p.tag = next_tag();
  p.err = device_error_word();
  for (int i = 0; i < 3; ++i) p.v_stride[i] = a.v_stride[i];
  p.table_stride = a.table_stride;
  p.requests = static_cast<int>(a.requests);
  p.tokens = static_cast<int>(a.tokens);
  p.heads = static_cast<int>(a.heads);
  p.kv_heads = static_cast<int>(a.kv_heads);
  p.group = p.heads / p.kv_heads;
  while ((1LL << p.page_shift) < a.page_size) ++p.page_shift;
  p.num_blocks = static_cast<int>(a.num_blocks);
  p.table_cols = static_cast<int>(a.table_cols);
  p.mask_words = static_cast<int>(a.mask_words);
  double scale = a.sm_scale;
  if (scale == 0.0) scale = 1.0 / std::sqrt(static_cast<double>(a.head_dim));
  p.scale_log2 = static_cast<float>(scale * 1.44269504088896340736);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Lengths lie on the device: the rows of a request, on average, choose the
  // kernel. Any choice is right for any lengths; a request with more rows than
  // a tile holds takes several and reads its keys for each. (8 requests x 1
  // token x 8 heads over 4096 keys: 17.6 us with the few-rows kernel, 23.6 with
  // this one; at 32 rows to a unit that kernel's softmax outgrows its
  // registers: 16 x 8 tokens x 4 heads 25 us for 16.)
  const int64_t rows = a.requests > 0 ? (a.tokens + a.requests - 1) / a.requests * p.group : p.group;
  cudaError_t e;
  if (rows <= kFewRows)
    e = launch_tree_few(p, a, s);
  else if (a.dtype == FL_DTYPE_F16)
    e = a.head_dim == 64 ? launch<__half, 64>(p, a, rows, s) : launch<__half, 128>(p, a, rows, s);
  else
    e = a.head_dim == 64 ? launch<__nv_bfloat16, 64>(p, a, rows, s) : launch<__nv_bfloat16, 128>(p, a, rows, s);
  return e == cudaSuccess ? FL_OK : cuda_fail(e, "tree attention launch");
}

}  // namespace

bool encode_tree_maps(TreeParams& p, const fl_tree_attention_args& a, int tile_keys) {
  const bool bf16 = a.dtype == FL_DTYPE_BF16;
  p.box_rows = static_cast<int>(std::min<int64_t>(a.page_size, tile_keys));
  const cuuint64_t dq[3] = {static_cast<cuuint64_t>(a.head_dim), static_cast<cuuint64_t>(a.heads),
                            static_cast<cuuint64_t>(a.tokens)};
  const cuuint64_t dc[4] = {static_cast<cuuint64_t>(a.head_dim), static_cast<cuuint64_t>(a.page_size),
                            static_cast<cuuint64_t>(a.kv_heads), static_cast<cuuint64_t>(a.num_blocks)};
  const int64_t sq[2] = {a.q_stride[1], a.q_stride[0]};
  const int64_t sk[3] = {a.k_stride[1], a.k_stride[2], a.k_stride[0]}, sv[3] = {a.v_stride[1], a.v_stride[2], a.v_stride[0]};
  const cuuint32_t bq[3] = {64, static_cast<cuuint32_t>(p.group), static_cast<cuuint32_t>(p.tile_tokens)};
  const cuuint32_t bc[4] = {64, static_cast<cuuint32_t>(p.box_rows), 1, 1};
  return encode(&p.tm_q, bf16, a.q, 3, dq, sq, bq) && encode(&p.tm_k, bf16, a.k_cache, 4, dc, sk, bc) &&
         encode(&p.tm_v, bf16, a.v_cache, 4, dc, sv, bc);
}

}  // namespace fl

extern "C" size_t fl_tree_attention_workspace_size(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  if (tokens <= 0 || heads <= 0 || kv_heads <= 0 || (head_dim != 64 && head_dim != 128)) return 0;
  if (!fl::prepare_current_device()) return 0;
  return fl::workspace_bytes(fl::kCtasPerSm * fl::sm_count(), head_dim);
}

extern "C" int fl_tree_attention(const fl_tree_attention_args* args, void* stream) {
  return fl::guarded([&] { return fl::tree_attention(args, stream); });
}
