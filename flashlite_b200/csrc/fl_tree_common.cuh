// Shared by the kernels of attention over a paged cache (fl_tree.cu: up to 128
// rows a unit; fl_tree_few.cu: few rows): launch parameters, the division of
// the work, the joining of cut units and the guard of V tiles.
//
// A unit of work is (request, key head, row tile): as many of the request's
// tokens as fill a tile's rows, each with the query heads that share the key
// head, so that a key and value is read once for all of them. A unit's keys
// are cut into tiles; all tiles of all units, laid end to end, are divided
// evenly among the CTAs whatever the requests' lengths, which are read on the
// device. A CTA that ends up with part of a unit leaves an fp32 partial
// result, and whichever CTA finishes a cut unit last joins its parts, in their
// order whoever that is (the same bits every time), and nobody waits for
// anyone.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/flashlite_b200.h"
#include "fl_internal.h"
#include "fl_ptx.cuh"
#include "fl_types.cuh"

namespace fl {

struct TreeParams {
  CUtensorMap tm_q;  // {D, heads, tokens}, box {64, group, tile_tokens}
  CUtensorMap tm_k;  // {D, page rows, key heads, blocks}, box {64, box_rows, 1, 1}
  CUtensorMap tm_v;
  const void* v;
  void* out;
  float* lse;
  const int32_t* table;
  const int32_t* context;
  const int32_t* cu;
  const uint32_t* mask;
  float* part;      // partial results, 2 * grid slots: CTA c's are 2c (a unit's later part) and 2c + 1 (its first)
  float2* part_sum; // their reference maximum (log2) and sum relative to it, a tile's rows for each slot
  unsigned long long* arrived;  // [2 * grid] by group of parts, [grid] by unit: tag and count
  unsigned long long tag;       // 48 bits, another one for each call
  unsigned int* err;
  long long v_stride[3];
  long long table_stride;
  int requests, tokens, heads, kv_heads, group, tile_tokens;
  int page_shift, box_rows, num_blocks, table_cols, mask_words;
  float scale_log2;
  int grid;
};

// Attention of few rows (fl_tree_few.cu): up to kFewRows to a unit. The caller
// has filled in everything but what depends on the kernel's tiles.
constexpr int kFewRows = 16;
cudaError_t launch_tree_few(TreeParams& p, const fl_tree_attention_args& a, cudaStream_t stream);
// Tensor maps of q, the caches for tiles of kBN keys and row tiles of p.tile_tokens.
bool encode_tree_maps(TreeParams& p, const fl_tree_attention_args& a, int tile_keys);

namespace {

constexpr int kSegRing = 3;  // work descriptors between the scheduler and the other warps

// A reference maximum is kept until a row's maximum exceeds it by this much
// (log2); probabilities are held 2^kUp times their size, so that fp16 keeps
// the small ones out of its subnormal range: at most 2^15 after the lag.
constexpr float kLag = 8.0f, kUp = 7.0f;

// One request as the schedule sees it.
struct Request {
  int begin, count, ctx, room;  // first row of q, new tokens, cached tokens, keys its table row can name
};

__device__ __forceinline__ Request request_of(const TreeParams& p, int begin, int end, int ctx, bool report) {
  Request r;
  const long long room = static_cast<long long>(p.table_cols) << p.page_shift;
  const bool part = ctx != -1;  // a request that takes no part (a refused one) sees no key
  if (!part) ctx = 0;
  r.room = !part ? 0 : room > 0x3fffffff ? 0x3fffffff : static_cast<int>(room);
  bool sound = true;
  r.begin = begin;
  r.count = end - begin;
  if (begin < 0 || end < begin || end > p.tokens) {
    sound = false;
    r.begin = r.count = 0;
  }
  r.ctx = ctx;
  if (ctx < 0 || ctx > r.room) {
    sound = false;
    r.ctx = ctx < 0 ? 0 : r.room;
  }
  if (part && r.count > r.room - r.ctx) sound = false;  // the new tokens past the table's end are not visible
  if (!sound && report) atomicOr(p.err, kDevErrIndex);
  return r;
}

// Keys that some row of the row tile with tokens [i0, i0 + n) may see.
__device__ __forceinline__ int keys_of(const TreeParams& p, const Request& r, int i0) {
  const int inner = p.mask != nullptr ? min(r.count, 32 * p.mask_words) : min(r.count, i0 + p.tile_tokens);
  return min(r.ctx + inner, r.room);
}

template <int kBN>
__device__ __forceinline__ int tiles_of(const TreeParams& p, const Request& r, int i0) {
  return max(1, (keys_of(p, r, i0) + kBN - 1) / kBN);
}

// Tiles of one key head of a request: those of all its row tiles, and `gap`
// more for each.
template <int kBN>
__device__ __forceinline__ long long head_tiles(const TreeParams& p, const Request& r, int gap) {
  if (r.count == 0) return 0;
  if (p.mask != nullptr)
    return static_cast<long long>((r.count + p.tile_tokens - 1) / p.tile_tokens) * (tiles_of<kBN>(p, r, 0) + gap);
  long long n = 0;
  for (int i0 = 0; i0 < r.count; i0 += p.tile_tokens) n += tiles_of<kBN>(p, r, i0) + gap;
  return n;
}

// a / b for a >= 0, b > 0. Not inlined: the scheduler divides in many places,
// once each, and on the path from a launch to its first load code that runs
// once costs what it takes to fetch (inlined with a fast path for small
// numbers, it made the smallest call 3 us longer).
__device__ __noinline__ long long divide(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// The division of `total` tiles among `used` CTAs: CTA c begins with tile
// floor(c total / used), so that tile u is the share of CTA
// ceil((u + 1) used / total) - 1.
struct Division {
  long long total, quot;
  int used, rem;
  __device__ __forceinline__ void init(long long total_, int grid) {
    total = total_;
    used = static_cast<int>(min(static_cast<long long>(grid), total));
    quot = used > 0 ? divide(total, used) : 0;
    rem = static_cast<int>(total - quot * used);
  }
  __device__ __forceinline__ long long begin(int c) const { return c * quot + divide(c * rem, used); }
  __device__ __forceinline__ int owner(long long u) const { return static_cast<int>(divide((u + 1) * used - 1, total)); }
};

// A CTA's share of one unit: tiles [t0, t1) of n.
struct Segment {
  int request, head, i0, rows;  // rows = tokens in the row tile times group
  int begin, ctx, keys;
  int t0, t1;                   // t1 < 0: no more work
  int slot;                     // partial result, -1: the whole unit, written to out
  int part, parts;              // which of the unit's how many parts
};


// The scheduler of one CTA: a warp that walks over the CTA's share of the
// tiles and hands out its segments. All lanes hold the same state, but for the
// 32 requests from `base` on, one a lane.
//
// kAligned: where a launch has fewer units than CTAs, every CTA takes at most
// one part of one unit, all parts of a unit are of one size and short units
// stay whole: joining costs 3 us on the way to the result, as much as
// kWholeTiles tiles. Parts at like places of neighbouring key heads run side
// by side, which read the same rows of memory where heads are interleaved. The
// division is taken where it is within an eighth of even (one cache of 131072
// keys, 8 heads: 56 us for 63) or its parts are short all the same (8 requests
// of up to 4096 keys: 16.7 us for 22.1, few cuts against many).
constexpr int kWholeTiles = 3, kShortPart = 8;

//
// kGap: the tiles that a change of units costs a CTA. Units are divided as if
// they began with so many more, so that CTAs with more units get fewer tiles.
template <int kBN, bool kAligned, int kGap>
struct Scheduler {
  const TreeParams& p;
  const int cta, lane;
  Division div;
  int part_tiles;        // aligned: tiles of a part; 0: even division
  int unit_tiles, unit_parts;  // aligned: those of the unit
  long long s, s1, off;  // next tile, end of the share, tiles of the current request before s
  int b, h, i0;          // request, key head, first token of the row tile
  bool entered;          // whether h and i0 are those of request b
  int base, l_begin, l_end, l_ctx;
  Request r;

  // used = false: a warp that only has the object.
  __device__ __forceinline__ Scheduler(const TreeParams& p_, int cta_, int lane_, bool used = true)
      : p(p_), cta(cta_), lane(lane_) {
    if (!used) return;
    load(0);
    if constexpr (kAligned) {
      start();
      if (p.requests <= 32 && aligned()) return;
    }
    const int per = (p.requests + 31) / 32;  // each lane sums a run of requests
    const int b0 = min(lane * per, p.requests), b1 = min(b0 + per, p.requests);
    long long mine = 0;
    if (per <= 1) {
      if (lane < p.requests) mine = p.kv_heads * head_tiles<kBN>(p, request_of(p, l_begin, l_end, l_ctx, cta == 0), kGap);
    } else {
      for (int x = b0; x < b1; ++x) mine += tiles(x, cta == 0);
    }
    long long before = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, before, d);
      if (lane >= d) before += x;
    }
    div.init(__shfl_sync(0xffffffffu, before, 31), p.grid);
    before -= mine;
    start();
    if (cta >= div.used) return;
    s = div.begin(cta);
    s1 = div.begin(cta + 1);
    const bool here = before <= s && s < before + mine;  // the share begins in this lane's run
    if (here) {
      b = b0;
      if (per > 1) {
        for (long long n = tiles(b, false); s >= before + n; n = tiles(b, false)) {
          before += n;
          ++b;
        }
      }
      off = s - before;
    }
    const int owner = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    b = __shfl_sync(0xffffffffu, b, owner);
    off = __shfl_sync(0xffffffffu, off, owner);
  }

  __device__ __forceinline__ void start() {
    s = s1 = off = 0;
    b = h = i0 = 0;
    entered = false;
    part_tiles = 0;
  }
  __device__ __forceinline__ int parts_of(int n) const {
    if (n <= kWholeTiles || n <= part_tiles) return 1;
    return part_tiles == 1 ? n : static_cast<int>(static_cast<uint32_t>(n + part_tiles - 1) / part_tiles);
  }
  // Takes the aligned division, if it is to be taken, and finds part number
  // `cta` of all: request b (lane b), key head h, first token i0, tiles and
  // parts of the unit and, as s, the part's number within it. s1 = s: there is
  // none. A chain of dependent steps on the way to the first load, 3,100 cycles
  // with the loads of the lengths (5,700, and 1.4 us more on the smallest call,
  // by way of the even division): one request a lane, 32-bit numbers, no
  // division where it would be by one.
  __device__ __forceinline__ bool aligned() {
    const Request mine = request_of(p, l_begin, l_end, l_ctx, cta == 0);
    const bool one = mine.count <= p.tile_tokens;  // at most one row tile
    const int row_tiles = one ? min(mine.count, 1) : (mine.count + p.tile_tokens - 1) / p.tile_tokens;
    if (__any_sync(0xffffffffu, row_tiles > 1 << 10) || p.kv_heads > 1 << 10) return false;  // totals below 2^30
    const int units = __reduce_add_sync(0xffffffffu, row_tiles) * p.kv_heads;
    if (units >= p.grid) return false;
    const int first_tiles = tiles_of<kBN>(p, mine, 0);
    const long long tiles = one ? row_tiles * first_tiles : head_tiles<kBN>(p, mine, 0);
    if (__any_sync(0xffffffffu, tiles > 1 << 15)) return false;
    const int total = __reduce_add_sync(0xffffffffu, static_cast<int>(tiles)) * p.kv_heads;
    const int spare = p.grid - units;  // sum of ceil(n / part_tiles) <= grid
    const int m = total <= spare ? 1 : static_cast<int>(static_cast<uint32_t>(total + spare - 1) / spare);
    if (m > kShortPart && 8LL * m * p.grid > 9LL * total) return false;
    part_tiles = m;
    int per_head = one ? row_tiles * parts_of(first_tiles) : 0;
    if (!one)
      for (int i = 0; i < row_tiles; ++i) per_head += parts_of(tiles_of<kBN>(p, mine, i * p.tile_tokens));
    const int all = per_head * p.kv_heads;
    int upto = all;
    if (p.requests > 1) {
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += x;
      }
    }
    const uint32_t after = __ballot_sync(0xffffffffu, upto > cta);
    if (after == 0) return true;
    b = __ffs(after) - 1;
    int rest = cta - __shfl_sync(0xffffffffu, upto - all, b);
    r.begin = __shfl_sync(0xffffffffu, mine.begin, b);
    r.count = __shfl_sync(0xffffffffu, mine.count, b);
    r.ctx = __shfl_sync(0xffffffffu, mine.ctx, b);
    r.room = __shfl_sync(0xffffffffu, mine.room, b);
    const uint32_t ph = __shfl_sync(0xffffffffu, per_head, b);
    h = static_cast<int>(static_cast<uint32_t>(rest) / ph);
    rest -= h * ph;
    while (true) {
      unit_tiles = tiles_of<kBN>(p, r, i0);
      unit_parts = parts_of(unit_tiles);
      if (rest < unit_parts) break;
      rest -= unit_parts;
      i0 += p.tile_tokens;
    }
    s = rest;
    s1 = rest + 1;
    return true;
  }

  // The next segment, or t1 = -1 after the last.
  __device__ __forceinline__ Segment next() {
    Segment g = {};
    g.t1 = -1;
    if (s >= s1) return g;
    if (kAligned && part_tiles > 0) {
      fill(g);
      g.parts = unit_parts;
      g.part = static_cast<int>(s);
      // the first parts have one tile more where they do not come out even
      const int each = unit_parts == unit_tiles ? 1 : unit_parts == 1 ? unit_tiles : unit_tiles / unit_parts;
      const int more = unit_tiles - each * unit_parts;
      g.t0 = g.part * each + min(g.part, more);
      g.t1 = g.t0 + each + (g.part < more ? 1 : 0);
      g.slot = g.parts == 1 ? -1 : 2 * cta + (g.part == 0 ? 1 : 0);
      s1 = s;
      return g;
    }
    while (true) {
      if (!entered) {
        if (b >= p.requests) return g;
        if (b >= base + 32) load(b);
        r = request_of(p, __shfl_sync(0xffffffffu, l_begin, b - base), __shfl_sync(0xffffffffu, l_end, b - base),
                       __shfl_sync(0xffffffffu, l_ctx, b - base), false);
        h = i0 = 0;
        if (off > 0) {  // the share begins inside this request
          const long long per_head = head_tiles<kBN>(p, r, kGap);
          h = static_cast<int>(divide(off, per_head));
          off -= h * per_head;
          if (p.mask != nullptr) {
            const int n = tiles_of<kBN>(p, r, 0) + kGap, rt = static_cast<int>(divide(off, n));
            i0 = rt * p.tile_tokens;
            off -= static_cast<long long>(rt) * n;
          } else {  // 32 row tiles at a time
            while (true) {
              const int mine = i0 + lane * p.tile_tokens;
              int upto = mine < r.count ? tiles_of<kBN>(p, r, mine) + kGap : 0;
#pragma unroll
              for (int d = 1; d < 32; d <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += x;
              }
              const int skip = __popc(__ballot_sync(0xffffffffu, upto <= off));
              if (skip > 0) off -= __shfl_sync(0xffffffffu, upto, skip - 1);
              i0 += skip * p.tile_tokens;
              if (skip < 32) break;
            }
          }
        }
        entered = true;
      }
      if (i0 >= r.count) {
        i0 = 0;
        ++h;
      }
      if (r.count > 0 && h < p.kv_heads) break;
      ++b;
      off = 0;
      entered = false;
    }
    const int n = tiles_of<kBN>(p, r, i0);
    g.t0 = max(static_cast<int>(off) - kGap, 0);
    const int t1 = static_cast<int>(min(static_cast<long long>(n), off + (s1 - s) - kGap));
    if (kGap > 0 && t1 <= g.t0) {  // the share ends before the unit's first tile
      s = s1;
      return g;
    }
    g.t1 = t1;
    fill(g);
    const bool whole = g.t0 == 0 && g.t1 == n;
    g.slot = whole ? -1 : 2 * cta + (g.t0 == 0 ? 1 : 0);
    g.part = 0;
    g.parts = 1;
    if (!whole) {
      const long long tile0 = s - off + kGap;
      const int first = div.owner(tile0);
      g.part = cta - first;
      g.parts = div.owner(tile0 + n - 1) - first + 1;
    }
    s += g.t1 + kGap - off;
    off = 0;
    i0 += p.tile_tokens;
    return g;
  }

 private:
  __device__ __forceinline__ void fill(Segment& g) const {
    g.request = b;
    g.head = h;
    g.i0 = i0;
    g.rows = min(p.tile_tokens, r.count - i0) * p.group;
    g.begin = r.begin;
    g.ctx = r.ctx;
    g.keys = keys_of(p, r, i0);
  }
  __device__ __forceinline__ void load(int from) {
    base = from;
    const int x = from + lane;
    l_begin = l_end = l_ctx = 0;
    if (x < p.requests) {
      l_begin = p.cu[x];
      l_end = p.cu[x + 1];
      l_ctx = p.context[x];
    }
  }
  __device__ __forceinline__ long long tiles(int x, bool report) const {
    return p.kv_heads * head_tiles<kBN>(p, request_of(p, p.cu[x], p.cu[x + 1], p.context[x], report), kGap);
  }
};

// Block numbers of a segment's pages, for a producer warp: 32 at a time, one a
// lane, and the next 32 already under way. (Read one tile ahead, they arrived
// too late once the memory was busy.)
template <int kBN>
struct PageNumbers {
  const TreeParams& p;
  const int32_t* row;
  int base, last, cur, next, lane;

  __device__ __forceinline__ PageNumbers(const TreeParams& p_, const Segment& g, int lane_) : p(p_), lane(lane_) {
    row = p.table + g.request * p.table_stride;
    base = g.t0 * kBN >> p.page_shift;
    last = (min(g.t1 * kBN, g.keys) - 1) >> p.page_shift;  // -1: no key at all
    cur = load(base + lane);
    next = load(base + 32 + lane);
  }
  __device__ __forceinline__ void begin_tile(int t) {
    if ((t * kBN >> p.page_shift) - base >= 32) {
      cur = next;
      base += 32;
      next = load(base + 32 + lane);
    }
  }
  // Page boxes of tile t that hold visible keys.
  __device__ __forceinline__ int boxes(const Segment& g, int t) const {
    return (max(0, min(kBN, g.keys - t * kBN)) + p.box_rows - 1) / p.box_rows;
  }
  // The block with this lane's key; num_blocks (outside the map: zeros arrive
  // and nothing is read) for a number out of range.
  __device__ __forceinline__ int block(int key, bool live, bool report) const {
    const int blk = __shfl_sync(0xffffffffu, cur, (key >> p.page_shift) - base);
    if (blk >= 0 && blk < p.num_blocks) return blk;
    if (live && report) atomicOr(p.err, kDevErrIndex);
    return p.num_blocks;
  }

 private:
  __device__ __forceinline__ int load(int page) const { return page <= last ? row[page] : 0; }
};

// Warp `worker` of `workers` loads its share of tile t's page boxes into
// shared memory ([kBN][64-column halves]), completing on `bar`; a lane for
// each box. A copy takes its warp some 125 cycles to issue, however it is
// written, so that small pages want several warps.
template <int HD, int kBN>
__device__ __forceinline__ void load_tile(const TreeParams& p, const CUtensorMap* tm, const PageNumbers<kBN>& pages,
                                          const Segment& g, int t, uint32_t dst, uint32_t bar, int worker, int workers,
                                          bool report) {
  const int lane = pages.lane, n = pages.boxes(g, t);
  if (worker == 0) {
    if (lane == 0) mbar_arrive_expect_tx(bar, n * p.box_rows * 128 * (HD / 64));
    __syncwarp();
  }
  const int box = lane * workers + worker, key = t * kBN + box * p.box_rows;
  const bool live = box < n;
  const int blk = pages.block(key, live, report);
  if (live) {
#pragma unroll
    for (int hh = 0; hh < HD / 64; ++hh)
      tma_load_4d(dst + hh * (kBN * 128) + box * p.box_rows * 128, tm, bar, 64 * hh, key & ((1 << p.page_shift) - 1), g.head,
                  blk);
  }
  __syncwarp();
}

__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity, volatile int* abort_flag, unsigned int* err) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err));
}
__device__ __forceinline__ bool wait_all_issuer(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                                unsigned int* err) {
  return __all_sync(0xffffffffu, mbar_wait_issuer(bar, parity, abort_flag, err));
}

// Exponent bits of the type, all set in infinities and NaN.
template <typename T>
constexpr uint32_t kExpBits = 0x7C00u;
template <>
constexpr uint32_t kExpBits<__nv_bfloat16> = 0x7F80u;

// A pair with its infinite and NaN elements cleared.
template <typename T>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
  constexpr uint32_t e = kExpBits<T>;
  if ((w & e) == e) w &= 0xffff0000u;
  if ((w >> 16 & e) == e) w &= 0x0000ffffu;
  return w;
}
// acc + 0 * w: NaN from then on if an element of w is infinite or NaN.
__device__ __forceinline__ uint32_t taint(uint32_t acc, uint32_t w, __half) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&w), __half2half2(__ushort_as_half(0)),
                            *reinterpret_cast<const __half2*>(&acc));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t taint(uint32_t acc, uint32_t w, __nv_bfloat16) {
  const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w),
                                   __bfloat162bfloat162(__ushort_as_bfloat16(0)),
                                   *reinterpret_cast<const __nv_bfloat162*>(&acc));
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// Makes a V tile of [kBN][HD] (64-column halves side by side) safe for the
// product, by one warp: rows [valid, kBN) cleared, infinities and NaN in rows
// [mixed, valid) cleared. Returns whether any were.
template <typename T, int HD, int kBN>
__device__ __forceinline__ bool guard_v(uint32_t tile, int mixed, int valid, int lane) {
  uint32_t acc = 0;
#pragma unroll
  for (int hh = 0; hh < HD / 64; ++hh) {
    const uint32_t half = tile + hh * (kBN * 128);
    for (int c = valid * 8 + lane; c < kBN * 8; c += 32) st_shared_v4(half + c * 16, 0u, 0u, 0u, 0u);
    // a first look, in which a multiplication by zero finds what is not finite
#pragma unroll 4
    for (int c = mixed * 8 + lane; c < valid * 8; c += 32) {
      const uint4 v = ld_shared_v4(half + c * 16);
      acc = taint(taint(taint(taint(acc, v.x, T()), v.y, T()), v.z, T()), v.w, T());
    }
  }
  const bool bad = finite2<T>(acc) != acc;
  if (__any_sync(0xffffffffu, bad)) {
#pragma unroll 1
    for (int hh = 0; hh < HD / 64; ++hh) {
      const uint32_t half = tile + hh * (kBN * 128);
#pragma unroll 1
      for (int c = mixed * 8 + lane; c < valid * 8; c += 32) {
        const uint4 v = ld_shared_v4(half + c * 16);
        st_shared_v4(half + c * 16, finite2<T>(v.x), finite2<T>(v.y), finite2<T>(v.z), finite2<T>(v.w));
      }
    }
  }
  fence_proxy_async_smem();
  return __any_sync(0xffffffffu, bad);
}

// Parts are joined in groups of so many, and the groups' results once more.
// Few rows: up to 18 x 18 parts, one for each CTA, and no CTA reads more than
// 18 at once. With 128 rows a part is 64 KB and takes 1.5 us to join, so that
// from 8 parts on both steps are kept equally short (a request of 49 parts,
// 216 rows over 15445 keys: 48 us for 58).
constexpr int kJoinFew = 18, kJoinMany = 7;
// First part of g's group, if groups are of so many parts.
__device__ __forceinline__ int group_base(const Segment& g, int size) { return g.parts <= size ? 0 : g.part / size * size; }
__device__ __forceinline__ int join_group(const Segment& g) {
  if (g.rows <= 32) return kJoinFew;
  int n = kJoinMany;
  if (g.parts > n)
    for (n = 3; n * n < g.parts;) ++n;
  return n;
}

// Arrivals are counted in 64-bit words of the workspace: the call's tag above
// a 16-bit count. The memory needs no clearing: before its part is begun each
// CTA turns a word with another tag, whatever an earlier use left there, into
// this call's with a count of zero (one of them succeeds, and none can after
// the first arrival). The last arrival clears the word, for a captured call
// that runs again with the same tag.
__device__ __forceinline__ int slot_of(int first, int part) { return part == 0 ? 2 * first + 1 : 2 * (first + part); }
__device__ __forceinline__ unsigned long long* group_word(const TreeParams& p, const Segment& g, int cta, int size) {
  return p.arrived + slot_of(cta - g.part, group_base(g, size));
}
__device__ __forceinline__ unsigned long long* unit_word(const TreeParams& p, const Segment& g, int cta) {
  return p.arrived + 2 * p.grid + (cta - g.part);
}
// By the first two lanes of the scheduler warp, for a part g of CTA cta.
__device__ __forceinline__ void ready_counts(const TreeParams& p, const Segment& g, int cta, int lane, int size) {
  if (lane >= 2) return;
  unsigned long long* word = lane == 0 ? group_word(p, g, cta, size) : unit_word(p, g, cta);
  const unsigned long long seen = *reinterpret_cast<volatile unsigned long long*>(word);
  if ((seen >> 16) != p.tag) atomicCAS(word, seen, p.tag << 16);
}
__device__ __forceinline__ bool arrive_last(unsigned long long* word, int n) {
  unsigned long long old;
  asm volatile("atom.acq_rel.gpu.global.add.u64 %0, [%1], 1;" : "=l"(old) : "l"(word) : "memory");
  if (static_cast<int>(old & 0xffffu) + 1 != n) return false;
  *reinterpret_cast<volatile unsigned long long*>(word) = 0ull;
  return true;
}

// One step of a join, a running maximum over parts taken two (or more) at a
// time: acc, sum and m take in parts with references l.x, sums l.y and values v.
// (A part's log2-sum-exp in the place of the two would lose the sum where
// scores are large: at 2^24 parts of 64 keys and of 1 would weigh the same.)
template <int kBatch, int kVals>
__device__ __forceinline__ void join_step(float& m, float& sum, float (&acc)[kVals], const float2 (&l)[kBatch],
                                          const float (&v)[kBatch][kVals]) {
  float m_new = m;
#pragma unroll
  for (int k = 0; k < kBatch; ++k) m_new = fmaxf(m_new, l[k].x);
  const float m_use = m_new == -INFINITY ? 0.0f : m_new, alpha = ex2_approx(m - m_use);
  m = m_new;
  sum *= alpha;
#pragma unroll
  for (int j = 0; j < kVals; ++j) acc[j] *= alpha;
#pragma unroll
  for (int k = 0; k < kBatch; ++k) {
    const float w = ex2_approx(l[k].x - m_use) * l[k].y;
    sum += w;
#pragma unroll
    for (int j = 0; j < kVals; ++j) acc[j] = fmaf(w, v[k][j], acc[j]);
  }
}
__device__ __forceinline__ float join_inv(float sum) { return sum == 0.0f ? 0.0f : 1.0f / sum; }
__device__ __forceinline__ float join_lse(float m, float sum) { return sum == 0.0f ? -INFINITY : m + log2f(sum); }
__device__ __forceinline__ void get4(float* to, const float4& v) {
  to[0] = v.x;
  to[1] = v.y;
  to[2] = v.z;
  to[3] = v.w;
}

// Rows of q that belong to no request (a batch padded to a fixed size, offsets
// out of range) give 0 and -inf: by warp `worker` of `workers`, of those whose
// work ends before the epilogue's (by the softmax warps it made the smallest
// call 0.7 us longer). Where all offsets are in order these are the rows before
// the first request and after the last; else each token is looked for in every
// request.
template <typename T, int HD>
__device__ __forceinline__ void clear_padding(const TreeParams& p, int worker, int workers, int lane) {
  auto clear = [&](long long orow) {
    if (lane < HD / 8) reinterpret_cast<uint4*>(static_cast<T*>(p.out) + orow * HD)[lane] = make_uint4(0u, 0u, 0u, 0u);
    if (p.lse != nullptr && lane == 0) p.lse[orow] = -INFINITY;
  };
  auto sound = [&](int begin, int end) { return begin >= 0 && end >= begin && end <= p.tokens; };
  bool in_order = true;
#pragma unroll 4
  for (int b = lane; b < p.requests; b += 32) in_order &= sound(p.cu[b], p.cu[b + 1]);
  if (__all_sync(0xffffffffu, in_order)) {
    const int first = p.requests > 0 ? p.cu[0] : 0, end = p.requests > 0 ? p.cu[p.requests] : 0;
    const long long before = static_cast<long long>(first) * p.heads;
    const long long rows = before + static_cast<long long>(p.tokens - end) * p.heads;
    for (long long r = worker; r < rows; r += workers)
      clear(r < before ? r : static_cast<long long>(end) * p.heads + (r - before));
    return;
  }
#pragma unroll 1
  for (int t = worker; t < p.tokens; t += workers) {
    bool mine = false;
#pragma unroll 1
    for (int b = lane; b < p.requests; b += 32) {
      const int begin = p.cu[b], end = p.cu[b + 1];
      mine |= sound(begin, end) && begin <= t && t < end;
    }
    if (__any_sync(0xffffffffu, mine)) continue;
#pragma unroll 1
    for (int h = 0; h < p.heads; ++h) clear(static_cast<long long>(t) * p.heads + h);
  }
}

// Whether every other of the n parts has arrived, so that this CTA need not
// put its own into memory: then the word is cleared.
__device__ __forceinline__ bool others_arrived(unsigned long long* word, unsigned long long tag, int n) {
  unsigned long long v;
  asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(word) : "memory");
  if (v != (tag << 16 | static_cast<unsigned>(n - 1))) return false;
  *reinterpret_cast<volatile unsigned long long*>(word) = 0ull;
  return true;
}

}  // namespace
}  // namespace fl
