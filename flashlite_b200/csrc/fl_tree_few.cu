// Attention over a paged cache for few rows: up to 16 to a unit, the tokens of
// a request times the query heads that share a key head (decoding single
// tokens, small trees). Same mathematics and roundings as fl_tree.cu, except
// that O is divided by the sum of all probabilities as rounded (fl_tree.cu:
// by the sum, corrected for each tile's largest only; the threads here hold
// the rounded ones of all rows anyway).
//
// Bound by the keys and values read once from memory, and for small calls by
// latency. With S = Q K^T as a 128-row product, so few rows would leave one
// softmax warp of four with work, on one quarter of the SM. So the products
// are transposed:
//   S^T = K Q^T      A = K tile (128 keys), B = Q (16 rows)
//   O^T += V^T P^T   A = V tile, read MN-major, B = P^T
// A TMEM lane, and a softmax thread, is a key with all the rows' scores: a
// tile's softmax takes 550 cycles for 128 keys, 1,300 for 64 the other way.
// The row maximum would be a reduction across the CTA; instead every thread
// compares its scores with the rows' common reference, and only when one
// exceeds it by more than the lag (once a unit as a rule; one barrier with an
// OR tells) the maxima are formed. The row sums stay in each thread until the
// end. O^T has the head dimension along the lanes, so that a warp writes a
// row's neighbouring columns.
//
// Two CTAs per SM, as one alone left the SMs uneven (one cache of 131072 keys:
// 88 us for 57): two producer warps, of which one is the scheduler too, that
// stream Q, K and V through one ring of 96 KB, an MMA warp for each product,
// the softmax warpgroup. S, P and O are double-buffered. Measured: 64 requests
// of up to 8192 keys, 32 heads over 8 of 128, bf16: 197 us, 6.3 TB/s, 96 % of
// the measured copy rate; one request of 777 keys, 8 heads of 64: 9.9 us.

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <string>

#include "fl_tree_common.cuh"

namespace fl {
namespace {

constexpr int kThreads = 256;
constexpr int kBN = 128;  // keys per tile (UMMA M)
constexpr int kRows = kFewRows;  // rows per unit (UMMA N): a P^T row is 32 bytes, one 32-byte swizzle atom
static_assert(kRows == 16, "one 32-byte swizzle atom");
constexpr int kCtasPerSm = 2;
constexpr int kProducers = 2;  // warps 0 and 3
constexpr int kGapTiles = 2;   // what a change of units costs (256 requests of 500 keys: 84 us, 93 with none)
// Register split: 128 x 112 (producers, MMA) + 128 x 144 (softmax) = 256 x 128, the launch's total.
constexpr int kRegsProducer = 112, kRegsSoftmax = 144;

template <int HD>
struct Few {
  static_assert(HD == 64 || HD == 128, "head dimension 64 or 128");
  static constexpr int kHalves = HD / 64;
  static constexpr int kTileBytes = kBN * HD * 2;        // 16 / 32 KB
  static constexpr int kStages = 96 * 1024 / kTileBytes;  // K and V tiles in turn
  static constexpr int kQBytes = kRows * HD * 2;
  static constexpr int kPBytes = kBN * kRows * 2;
  static constexpr int kSmemQ = kStages * kTileBytes;      // 2 buffers
  static constexpr int kSmemP = kSmemQ + 2 * kQBytes;      // 2 buffers
  static constexpr int kSmemMisc = kSmemP + 2 * kPBytes;
  // Tile n of the stream (K tiles even, V tiles odd) lies in stage n % kStages.
  // With an odd number of stages one stage holds K and V tiles in turn, whose
  // arrivals different warps wait for: they take barriers in turn too, since a
  // warp that waits for every other phase of a barrier takes the phase before
  // the one between for its own.
  static constexpr int kFull = kStages % 2 == 0 ? kStages : 2 * kStages;
  static __device__ __forceinline__ uint32_t full(uint32_t bar_full, int n) { return bar_full + 8 * (n % kFull); }
  static __device__ __forceinline__ uint32_t full_phase(int n) { return (n / kFull) & 1; }
  // barriers | segments | maxima [4][kRows] or sums [4][kRows][2] | 1 / sum [kRows] | flags
  static constexpr int kBars = kFull + kStages + 2 * kSegRing + 2 * 9 + 1;
  static constexpr int kOffSeg = (kBars * 8 + 15) / 16 * 16;
  static constexpr int kOffMax = kOffSeg + kSegRing * static_cast<int>(sizeof(Segment));
  static constexpr int kOffSum = kOffMax;  // never in use at the same time: a barrier lies between
  static constexpr int kOffInv = kOffMax + 8 * kRows * 4;
  static constexpr int kOffFlag = kOffInv + kRows * 4;
  static constexpr int kSmemBytes = kSmemMisc + kOffFlag + 20;
  static_assert(kOffMax % 16 == 0, "maxima are read four at a time");
  static_assert(kCtasPerSm * (kSmemBytes + 1024) <= 228 * 1024, "shared memory");
  static constexpr uint32_t kTmemCols = 4 * kRows;            // S, O: two buffers of kRows columns each
};

__device__ __forceinline__ uint64_t make_sdesc_p(uint32_t saddr) {
  constexpr uint64_t kLayout32 = 6;  // 32-byte swizzle
  const uint64_t d = make_sdesc_sw128(saddr, 16, kRows * 2 * 8);
  return (d & ~(7ull << 61)) | kLayout32 << 61;
}

__device__ __forceinline__ void tmem_ld_rows(uint32_t addr, uint32_t (&r)[kRows]) {
  tmem_ld16_nowait(addr, r);
  tmem_wait_ld16_dep(r);
}

// Barrier of the 128 softmax threads that also tells whether any had `x`.
__device__ __forceinline__ bool softmax_any(bool x) {
  uint32_t out;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(out)
      : "r"(static_cast<uint32_t>(x))
      : "memory");
  return out != 0;
}
__device__ __forceinline__ void softmax_sync() { named_bar_sync(1, 128); }

// Maximum over a warp; NaN does not take part.
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

// Sums over a warp of kRows values per lane: lanes 2 r and 2 r + 1 end with
// that of row r. Each step halves the values: 16 shuffles, not 80.
__device__ __forceinline__ float warp_sums(float (&a)[kRows], int lane) {
#pragma unroll
  for (int half = kRows / 2, d = 16; half > 0; half /= 2, d /= 2) {
    const bool up = lane & d;
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float send = up ? a[i] : a[i + half], keep = up ? a[i + half] : a[i];
      a[i] = keep + __shfl_xor_sync(0xffffffffu, send, d);
    }
  }
  return a[0] + __shfl_xor_sync(0xffffffffu, a[0], 1);
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) tree_few_kernel(const __grid_constant__ TreeParams p) {
  using C = Few<HD>;
  constexpr int kStages = C::kStages;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  const uint32_t s_q = sbase + C::kSmemQ, s_p = sbase + C::kSmemP;
  uint8_t* misc = smem + C::kSmemMisc;
  const uint32_t bars = sbase + C::kSmemMisc;
  const uint32_t bar_full = bars, bar_empty = bar_full + 8 * C::kFull;
  const uint32_t bar_segfull = bar_empty + 8 * kStages, bar_segempty = bar_segfull + 8 * kSegRing;
  // pairs: by segment (Q loaded, Q free, O read, V guard's finding) or by tile (the others)
  const uint32_t bar_qfull = bar_segempty + 8 * kSegRing, bar_qfree = bar_qfull + 16, bar_s = bar_qfree + 16,
                 bar_sfree = bar_s + 16, bar_p = bar_sfree + 16, bar_pv = bar_p + 16, bar_ofree = bar_pv + 16,
                 bar_seg = bar_ofree + 16, bar_count = bar_seg + 16, bar_drain = bar_count + 16;
  Segment* segs = reinterpret_cast<Segment*>(misc + C::kOffSeg);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc + C::kOffFlag);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + C::kOffFlag + 4);
  volatile int* last_flag = reinterpret_cast<volatile int*>(misc + C::kOffFlag + 8);
  volatile int* bad_flag = reinterpret_cast<volatile int*>(misc + C::kOffFlag + 12);  // two, by segment
  float* s_max = reinterpret_cast<float*>(misc + C::kOffMax);
  float* s_sum = reinterpret_cast<float*>(misc + C::kOffSum);
  float* s_inv = reinterpret_cast<float*>(misc + C::kOffInv);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x;

  // ---- setup, before the kernel ahead has finished ----
  if (tid == 0) {
    for (int i = 0; i < C::kFull; ++i) mbar_init(bar_full + 8 * i, 1);
    for (int i = 0; i < kStages; ++i) mbar_init(bar_empty + 8 * i, 1);
    for (int i = 0; i < kSegRing; ++i) {
      mbar_init(bar_segfull + 8 * i, 1);
      mbar_init(bar_segempty + 8 * i, 7);  // the other producer, two MMA warps and four softmax warps
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_qfull + 8 * i, 1);
      mbar_init(bar_qfree + 8 * i, 1);
      mbar_init(bar_s + 8 * i, 1);
      mbar_init(bar_sfree + 8 * i, 4);  // one arrival per softmax warp
      mbar_init(bar_p + 8 * i, 4);
      mbar_init(bar_pv + 8 * i, 1);
      mbar_init(bar_ofree + 8 * i, 4);
      mbar_init(bar_seg + 8 * i, 1);
      mbar_init(bar_count + 8 * i, 1);
    }
    mbar_init(bar_drain, 2);  // both MMA warps
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.tm_q);
    tma_prefetch_desc(&p.tm_k);
    tma_prefetch_desc(&p.tm_v);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kRegsProducer));
  if (warp == 0 || warp == 3) {
    // ======================= producers; warp 0 is the scheduler too =======================
    // (Between a launch and its first load there is no hand-over.)
    const int worker = warp == 0 ? 0 : 1;
    Scheduler<kBN, true, kGapTiles> sched(p, cta, lane, warp == 0);
    int n = 0, seg = 0;   // tiles of K and V, and Q tiles, so far
    uint32_t issued = 0;  // bit i: this warp has copies in tile n - 1 - i
    bool ok = true;
    while (ok) {
      const int sl = seg % kSegRing;
      Segment g;
      if (worker == 0) {
        g = sched.next();
      } else {
        if (!wait_all(bar_segfull + 8 * sl, (seg / kSegRing) & 1, abort_flag, p.err)) break;
        g = segs[sl];
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_segempty + 8 * sl);
      }
      PageNumbers<kBN> pages(p, g, lane);  // of none after the last segment
      if (worker == 0) {
        if (!wait_all(bar_segempty + 8 * sl, ((seg / kSegRing) & 1) ^ 1, abort_flag, p.err)) break;
        if (lane == 0) {
          segs[sl] = g;
          mbar_arrive(bar_segfull + 8 * sl);
        }
        __syncwarp();
      }
      if (g.t1 < 0) break;
      if (worker == 0) {
        if (!wait_all(bar_qfree + 8 * (seg & 1), ((seg >> 1) & 1) ^ 1, abort_flag, p.err)) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(bar_qfull + 8 * (seg & 1), p.group * p.tile_tokens * 128 * C::kHalves);
#pragma unroll
          for (int hh = 0; hh < C::kHalves; ++hh)
            tma_load_3d(s_q + (seg & 1) * C::kQBytes + hh * (kRows * 128), &p.tm_q, bar_qfull + 8 * (seg & 1), 64 * hh,
                        g.head * p.group, g.begin + g.i0);
        }
        __syncwarp();
      }
      ++seg;
      for (int t = g.t0; ok && t < g.t1; ++t) {
        pages.begin_tile(t);
        if (worker > 0 && pages.boxes(g, t) <= worker) {
          // No box of the tile is this warp's: it comes and goes without it. A
          // wait for its stage could find it used and freed already, and take
          // the phase it waits for for one still to come.
          n += 2;
          issued <<= 2;
          continue;
        }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++n) {
          const int st = n % kStages;
          if (!wait_all(bar_empty + 8 * st, ((n / kStages) & 1) ^ 1, abort_flag, p.err)) {
            ok = false;
            break;
          }
          load_tile<HD, kBN>(p, kv ? &p.tm_v : &p.tm_k, pages, g, t, sbase + st * C::kTileBytes, C::full(bar_full, n), worker,
                             kProducers, kv == 0);
          issued = issued << 1 | 1u;
        }
        if (worker == 0 && t == g.t0 && g.slot >= 0) {  // while the first tile is on its way
          ready_counts(p, g, cta, lane, kJoinFew);
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_count + 8 * (g.slot & 1));
        }
      }
    }
    if (*abort_flag && lane == 0) {
      // Let every copy that this warp started land before shared memory is
      // released. A stage is loaded anew only after its tile has come, but the
      // second warp may have skipped a tile (two of the stream) that the first
      // has yet to load.
      constexpr int kUnderWay = kStages + 2;
      static_assert(kUnderWay <= 32, "a bit for each");
      for (int i = max(n - kUnderWay, 0); i < n; ++i)
        if (issued >> (n - 1 - i) & 1u) mbar_wait_quiet(C::full(bar_full, i), C::full_phase(i));
      if (worker == 0)
        for (int i = max(seg - 2, 0); i < seg; ++i) mbar_wait_quiet(bar_qfull + 8 * (i & 1), (i >> 1) & 1);
    }
    __syncwarp();
    if (worker > 0) clear_padding<T, HD>(p, cta, p.grid, lane);
  } else if (warp == 1) {
    // ======================= S^T = K Q^T =======================
    constexpr uint32_t idesc = make_idesc_f16_f32(kBN, kRows, false, false, kBf16);  // K-major A (K) and B (Q)
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t dk0 = make_sdesc_sw128(sbase, 16, 1024), dq0 = make_sdesc_sw128(s_q, 16, 1024);
    constexpr uint64_t kTileEnc = C::kTileBytes >> 4, kKHalf = (kBN * 128) >> 4, kQHalf = (kRows * 128) >> 4;
    int js = 0, seg = 0;
    bool ok = true;
    while (ok) {
      const int sl = seg % kSegRing, i = seg & 1;
      if (!wait_all_issuer(bar_segfull + 8 * sl, (seg / kSegRing) & 1, abort_flag, p.err)) break;
      const int tiles = __shfl_sync(0xffffffffu, segs[sl].t1 - segs[sl].t0, 0);
      const bool done = segs[sl].t1 < 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_segempty + 8 * sl);
      if (done) break;
      if (!wait_all_issuer(bar_qfull + 8 * i, (seg >> 1) & 1, abort_flag, p.err)) break;
      for (int t = 0; t < tiles; ++t, ++js) {
        const int st = (2 * js) % kStages;  // K tiles are every other one of the stream
        if (!(ok = wait_all_issuer(C::full(bar_full, 2 * js), C::full_phase(2 * js), abort_flag, p.err))) break;
        if (!(ok = wait_all_issuer(bar_sfree + 8 * (js & 1), ((js >> 1) & 1) ^ 1, abort_flag, p.err))) break;
        tc_fence_after();
        const uint64_t ad = dk0 + st * kTileEnc, bd = dq0 + i * static_cast<uint64_t>(C::kQBytes >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            umma_f16_ss(tm + (js & 1) * kRows, ad + 2 * (kk & 3) + (kk >> 2) * kKHalf, bd + 2 * (kk & 3) + (kk >> 2) * kQHalf,
                        idesc, kk > 0 ? 1u : 0u);
          umma_commit(bar_s + 8 * (js & 1));
          umma_commit(bar_empty + 8 * st);
          if (t + 1 == tiles) umma_commit(bar_qfree + 8 * i);
        }
        __syncwarp();
      }
      ++seg;
    }
    // wait until every MMA this warp issued has completed
    if (elect_one()) {
      umma_commit(bar_drain);
      mbar_wait_quiet(bar_drain, 0);
    }
    __syncwarp();
  } else {
    // ======================= O^T += V^T P^T (warp 2) =======================
    // A warp of its own: it never holds a V tile while it waits for the next K
    // tile, and either product goes out as soon as it can.
    constexpr uint32_t idesc = make_idesc_f16_f32(kBN, kRows, true, true, kBf16);  // MN-major A (V) and B (P)
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    // 64-column halves of V one leading offset apart. With head dimension 64
    // the product's rows 64-127 are whatever lies there: not looked at.
    const uint64_t dv0 = make_sdesc_sw128(sbase, HD == 64 ? 8192 : kBN * 128, 1024), dp0 = make_sdesc_p(s_p);
    constexpr uint64_t kTileEnc = C::kTileBytes >> 4;
    int js = 0, seg = 0;
    bool ok = true;
    while (ok) {
      const int sl = seg % kSegRing, o = seg & 1;
      if (!wait_all_issuer(bar_segfull + 8 * sl, (seg / kSegRing) & 1, abort_flag, p.err)) break;
      const Segment g = segs[sl];
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_segempty + 8 * sl);
      if (g.t1 < 0) break;
      // O of the segment before the last has been read
      if (!wait_all_issuer(bar_ofree + 8 * o, ((seg >> 1) & 1) ^ 1, abort_flag, p.err)) break;
      if (lane == 0) bad_flag[o] = 0;
      // keys from here on are hidden from some row of the tile
      const int mixed = p.mask != nullptr ? g.ctx : min(g.ctx + g.i0 + 1, g.keys);
      uint32_t accumulate = 0;
      for (int t = g.t0; t < g.t1; ++t, ++js) {
        const int st = (2 * js + 1) % kStages;
        if (!(ok = wait_all_issuer(C::full(bar_full, 2 * js + 1), C::full_phase(2 * js + 1), abort_flag, p.err))) break;
        const int valid = min(kBN, g.keys - t * kBN), from = max(0, min(mixed - t * kBN, valid));
        if (from < kBN) {
          const bool bad = guard_v<T, HD, kBN>(sbase + st * C::kTileBytes, from, valid, lane);
          if (bad && lane == 0) bad_flag[o] = 1;
          __syncwarp();
        }
        if (!(ok = wait_all_issuer(bar_p + 8 * (js & 1), (js >> 1) & 1, abort_flag, p.err))) break;
        tc_fence_after();
        const uint64_t ad = dv0 + st * kTileEnc, bd = dp0 + (js & 1) * static_cast<uint64_t>(C::kPBytes >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kBN / 16; ++kk)
            umma_f16_ss(tm + 2 * kRows + o * kRows, ad + 128 * kk, bd + kk * (kRows * 2 * 16 >> 4), idesc, kk > 0 ? 1u : accumulate);
          umma_commit(bar_pv + 8 * (js & 1));
          umma_commit(bar_empty + 8 * st);
        }
        __syncwarp();
        accumulate = 1;
      }
      if (lane == 0) mbar_arrive(bar_seg + 8 * o);  // publishes bad_flag
      __syncwarp();
      ++seg;
    }
    if (elect_one()) {
      umma_commit(bar_drain);
      mbar_wait_quiet(bar_drain, 0);
    }
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kRegsSoftmax));
    // ======================= softmax: one thread per key =======================
    const int t_key = tid - 128;  // also the column of O this thread holds
    const uint32_t lane_base = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const float sc = p.scale_log2;
    // this thread's key in a P buffer: kRows elements, 16-byte chunks swizzled as the product reads them
    const uint32_t p_row = s_p + t_key * (kRows * 2);
    const int swz = (t_key >> 2) & 1;
    // Reference of a row that has seen nothing: no finite score is below it
    // (-infinity would turn hidden scores into NaN).
    constexpr float kNone = -FLT_MAX;
    int js = 0, seg = 0;               // tiles and segments so far
    // A wait that gives up clears ok. The four warps meet at barriers, so none
    // may leave alone: they look at each other's ok where they meet.
    bool ok = true;
    while (true) {
      const int sl = seg % kSegRing;
      ok = ok && wait_all(bar_segfull + 8 * sl, (seg / kSegRing) & 1, abort_flag, p.err);
      if (softmax_any(!ok)) break;
      const Segment g = segs[sl];
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_segempty + 8 * sl);
      if (g.t1 < 0) break;
      const uint32_t all_rows = g.rows >= 32 ? 0xffffffffu : (1u << g.rows) - 1u;
      const uint32_t tO = tmem + lane_base + 2 * kRows + (seg & 1) * kRows;
      // rows of the tile that see new token j of the request
      auto rows_seeing = [&](int j) -> uint32_t {
        if (p.mask == nullptr) {
          const int first = max(j - g.i0, 0) * p.group;  // rows of the tokens from j on
          return first >= 32 ? 0u : all_rows & ~((1u << first) - 1u);
        }
        uint32_t seen = 0;
        if ((j >> 5) < p.mask_words)
          for (int i = 0, r = 0; r < g.rows; ++i, r += p.group)
            if (p.mask[static_cast<long long>(g.begin + g.i0 + i) * p.mask_words + (j >> 5)] >> (j & 31) & 1u)
              seen |= (p.group >= 32 ? 0xffffffffu : (1u << p.group) - 1u) << r;
        return seen & all_rows;
      };
      float ref[kRows], l[kRows], lr[kRows];  // reference maxima less kUp; sums of p, and of p as rounded for the product
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        ref[r] = kNone;
        l[r] = lr[r] = 0.0f;
      }
      for (int t = g.t0; t < g.t1; ++t, ++js) {
        const int buf = js & 1;
        const int key = t * kBN + t_key;
        const uint32_t vis = key < g.ctx ? (key < g.keys ? all_rows : 0u) : key < g.keys ? rows_seeing(key - g.ctx) : 0u;
        ok = ok && wait_all(bar_s + 8 * buf, (js >> 1) & 1, abort_flag, p.err);
        tc_fence_after();
        uint32_t sr[kRows];
        tmem_ld_rows(tmem + lane_base + buf * kRows, sr);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_sfree + 8 * buf);
        // Scaled first: a fused multiply-add against a rounded reference could
        // be off by more than the lag where scores are large.
        float y[kRows], most = -INFINITY;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          y[r] = (vis >> r & 1u) ? __uint_as_float(sr[r]) * sc : -INFINITY;
          most = fmaxf(most, y[r] - ref[r]);
        }
        if (softmax_any(most > kLag + kUp || !ok)) {
          if (softmax_any(!ok)) {
            ok = false;
            break;
          }
          // new maxima: over the warp, then the four warps
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            if (r % 4 == 0 && r >= g.rows) break;  // four rows at a time: the others see nothing
            const float m = warp_max(y[r]);
            if (lane == 0) s_max[4 * r + (warp & 3)] = m;
          }
          softmax_sync();
          float alpha[kRows];
#pragma unroll
          for (int r = 0; r < kRows; ++r) alpha[r] = 1.0f;
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            if (r % 4 == 0 && r >= g.rows) break;
            const float4 w = reinterpret_cast<const float4*>(s_max)[r];
            const float m = fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w));
            const float next = m - ref[r] > kLag + kUp ? m - kUp : ref[r];
            alpha[r] = ex2_approx(ref[r] - next);  // 1, or 0 after kNone
            ref[r] = next;
            l[r] *= alpha[r];
            lr[r] *= alpha[r];
          }
          if (t > g.t0) {  // O takes the new reference when the last P V is in it
            ok = wait_all(bar_pv + 8 * (buf ^ 1), ((js - 1) >> 1) & 1, abort_flag, p.err);
            tc_fence_after();
            uint32_t o[kRows];
            tmem_ld_rows(tO, o);
#pragma unroll
            for (int r = 0; r < kRows; ++r) o[r] = __float_as_uint(__uint_as_float(o[r]) * alpha[r]);
            tmem_st16(tO, o);
            tmem_st_wait();
            tc_fence_before();
          }
        }
        uint32_t pk[kRows / 2];
#pragma unroll
        for (int r = 0; r < kRows; r += 2) {
          const float a = ex2_approx(y[r] - ref[r]), b = ex2_approx(y[r + 1] - ref[r + 1]);
          l[r] += a;
          l[r + 1] += b;
          pk[r / 2] = pack2<T>(a, b);
          const float2 f = unpack2<T>(pk[r / 2]);
          lr[r] += f.x;
          lr[r + 1] += f.y;
        }
        // the P V that read this buffer two tiles ago is done
        if (js >= 2) ok = ok && wait_all(bar_pv + 8 * buf, ((js >> 1) & 1) ^ 1, abort_flag, p.err);
#pragma unroll
        for (int c = 0; c < kRows / 8; ++c)
          st_shared_v4(p_row + buf * C::kPBytes + ((c ^ swz) << 4), pk[4 * c], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(bar_p + 8 * buf);
      }
      if (softmax_any(!ok)) break;

      // ---- epilogue of the segment: row sums, then O ----
      {
        const float sum = warp_sums(l, lane), sum_r = warp_sums(lr, lane);
        const int r = lane >> 1;
        if ((lane & 1) == 0) {
          s_sum[((warp & 3) * kRows + r) * 2] = sum;
          s_sum[((warp & 3) * kRows + r) * 2 + 1] = sum_r;
        }
      }
      softmax_sync();
      float sum = 0.0f, m = 0.0f;
      if (t_key < g.rows) {
        float sum_r = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          sum += s_sum[(w * kRows + t_key) * 2];
          sum_r += s_sum[(w * kRows + t_key) * 2 + 1];
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) m = r == t_key ? ref[r] : m;
        s_inv[t_key] = sum == 0.0f ? 0.0f : 1.0f / sum_r;
      }
      softmax_sync();
      if (t_key < g.rows) {
        if (g.slot >= 0)
          p.part_sum[g.slot * kRows + t_key] = make_float2(m, sum);
        else if (p.lse != nullptr)
          p.lse[static_cast<long long>(g.begin + g.i0 + t_key / p.group) * p.heads + g.head * p.group + t_key % p.group] =
              join_lse(m, sum) * 0.69314718055994531f;
      }
      ok = wait_all(bar_pv + 8 * ((js - 1) & 1), ((js - 1) >> 1) & 1, abort_flag, p.err) &&
           wait_all(bar_seg + 8 * (seg & 1), (seg >> 1) & 1, abort_flag, p.err);
      tc_fence_after();
      const bool bad = bad_flag[seg & 1] != 0;
      if (32 * (warp & 3) < HD) {
        uint32_t sr[kRows];
        tmem_ld_rows(tO, sr);
        float o[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) o[r] = r < g.rows ? __uint_as_float(sr[r]) * s_inv[r] : 0.0f;
        if (bad) {
          // infinities and NaN that guard_v cleared, for the rows that see them
          const int hidden = p.mask != nullptr ? g.ctx : g.ctx + g.i0 + 1;
          for (int key = max(hidden, g.t0 * kBN); key < min(g.t1 * kBN, g.keys); ++key) {
            const int blk = p.table[g.request * p.table_stride + (key >> p.page_shift)];
            if (blk < 0 || blk >= p.num_blocks) continue;
            const float x = static_cast<float>(static_cast<const T*>(p.v)[
                blk * p.v_stride[0] + (key & ((1 << p.page_shift) - 1)) * p.v_stride[1] + g.head * p.v_stride[2] + t_key]);
            if (fabsf(x) < INFINITY) continue;
            const uint32_t seen = rows_seeing(key - g.ctx);
#pragma unroll
            for (int r = 0; r < kRows; ++r)
              if (seen >> r & 1u) o[r] += x;
          }
        }
        if (g.slot >= 0) {
          float* to = p.part + static_cast<long long>(g.slot) * kRows * HD + t_key;
#pragma unroll
          for (int r = 0; r < kRows; ++r)
            if (r < g.rows) to[r * HD] = o[r];
        } else {
          T* to = static_cast<T*>(p.out) +
                  (static_cast<long long>(g.begin + g.i0) * p.heads + g.head * p.group) * HD + t_key;
          const long long next_token = static_cast<long long>(p.heads - p.group) * HD;
          int left = p.group;
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            if (r >= g.rows) break;
            *to = static_cast<T>(o[r]);
            to += HD;
            if (--left == 0) {
              left = p.group;
              to += next_token;
            }
          }
        }
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_ofree + 8 * (seg & 1));
      ++seg;

      if (g.slot >= 0) {
        // a part: whoever arrives last joins, within its group of parts and then among the groups:
        //   o = sum_k l_k 2^(m_k - M) o_k / sum_k l_k 2^(m_k - M),  M = max_k m_k
        const int first = cta - g.part, groups = (g.parts + kJoinFew - 1) / kJoinFew;
        int base = group_base(g, kJoinFew), stride = 1, n = min(kJoinFew, g.parts - base);
#pragma unroll 1
        while (true) {
          __syncwarp();
          if (softmax_any(!ok)) break;  // otherwise all of this CTA's part is written
          if (t_key == 0)
            *last_flag = mbar_wait(bar_count + 8 * (g.slot & 1), 0, abort_flag, p.err) &&
                         arrive_last(stride == 1 ? group_word(p, g, cta, kJoinFew) : unit_word(p, g, cta), n);
          softmax_sync();
          if (*last_flag == 0) break;
          const int to = stride == 1 && groups > 1 ? slot_of(first, base) : -1;
          constexpr int kVecs = HD / 4, kBatch = 9;
#pragma unroll 1
          for (int i = t_key; i < g.rows * kVecs; i += 128) {
            const int r = i / kVecs, c = i % kVecs;
            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            m = -INFINITY;
            sum = 0.0f;
#pragma unroll 1
            for (int k0 = 0; k0 < n; k0 += kBatch) {
              float2 l2[kBatch];
              float v[kBatch][4];
#pragma unroll
              for (int k = 0; k < kBatch; ++k) {
                const bool in = k0 + k < n;
                const int sl = slot_of(first, base + min(k0 + k, n - 1) * stride);
                l2[k] = in ? __ldcg(p.part_sum + sl * kRows + r) : make_float2(-INFINITY, 0.0f);
                get4(v[k], in ? __ldcg(reinterpret_cast<const float4*>(p.part + (static_cast<long long>(sl) * kRows + r) * HD) + c)
                              : make_float4(0.f, 0.f, 0.f, 0.f));
              }
              join_step<kBatch, 4>(m, sum, acc, l2, v);
            }
            const float inv = join_inv(sum);
            const float4 o = make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
            if (to >= 0) {
              reinterpret_cast<float4*>(p.part + (static_cast<long long>(to) * kRows + r) * HD)[c] = o;
              if (c == 0) reinterpret_cast<float2*>(s_sum)[r] = make_float2(m, sum);
            } else {
              const long long orow = static_cast<long long>(g.begin + g.i0 + r / p.group) * p.heads + g.head * p.group + r % p.group;
              reinterpret_cast<uint2*>(static_cast<T*>(p.out) + orow * HD)[c] = make_uint2(pack2<T>(o.x, o.y), pack2<T>(o.z, o.w));
              if (c == 0 && p.lse != nullptr) p.lse[orow] = join_lse(m, sum) * 0.69314718055994531f;
            }
          }
          if (to >= 0) {  // the group's sums have been read: its first slot takes the joined ones
            softmax_sync();
            if (t_key < g.rows) p.part_sum[to * kRows + t_key] = reinterpret_cast<const float2*>(s_sum)[t_key];
          }
          if (to < 0) break;
          base = 0;
          stride = kJoinFew;
          n = groups;
        }
      }
    }
  }

  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

template <typename T, int HD>
cudaError_t launch(TreeParams& p, cudaStream_t stream) {
  auto kern = tree_few_kernel<T, HD>;
  static std::atomic<bool> configured[kMaxFlagDevices];
  const cudaError_t e = ensure_smem_limit(kern, Few<HD>::kSmemBytes, configured);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, p.grid, kThreads, Few<HD>::kSmemBytes, stream, p);
}

}  // namespace

cudaError_t launch_tree_few(TreeParams& p, const fl_tree_attention_args& a, cudaStream_t stream) {
  p.grid = kCtasPerSm * sm_count();
  p.tile_tokens = kRows / p.group;
  p.part_sum = reinterpret_cast<float2*>(p.part + 2LL * p.grid * kRows * a.head_dim);
  p.arrived = reinterpret_cast<unsigned long long*>(p.part_sum + 2LL * p.grid * kRows);
  if (!encode_tree_maps(p, a, kBN)) return cudaErrorInvalidValue;
  if (a.dtype == FL_DTYPE_F16) return a.head_dim == 64 ? launch<__half, 64>(p, stream) : launch<__half, 128>(p, stream);
  return a.head_dim == 64 ? launch<__nv_bfloat16, 64>(p, stream) : launch<__nv_bfloat16, 128>(p, stream);
}

}  // namespace fl
