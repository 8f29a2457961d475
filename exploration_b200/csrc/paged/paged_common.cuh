// Shared pieces of the paged-cache attention kernels: the argument block, the
// split of the work over the CTAs of a launch, and the partial results that
// the combine kernel joins.
//
// A cache is a pool of pages [pages, kv_heads, page, dim]; `tables[b, j]`
// names the pool page with the keys of positions [j * page, (j + 1) * page) of
// sequence b. Query heads h * group .. h * group + group - 1 share key head h,
// so the rows of one (sequence, key head) are row r = token * group + g. A
// group larger than a kernel's row tile is divided into several items of the
// same key head.
//
// Work split. An entry is a (sequence, row tile); its key limit is one more
// than the largest position among its rows, so nothing but `positions` (on
// the device) says how long a sequence is: one captured launch serves every
// later step. The key tiles of all (entry, key head) items form one list, cut
// into equal runs, one a CTA: sequences of very different lengths and a few
// rows over a long cache both fill the GPU. Each item counts a few tiles more, for
// its start and end (with tiles alone the CTA that got fifteen short items of a
// ragged chunk took 409 us, most others 340). An item inside one run is written
// out by its CTA; an item that is cut leaves unnormalised partial sums (at most
// two a CTA: its first and its last item), which the combine kernel joins in
// key order, so results do not depend on the order in which CTAs finish. Each
// CTA notes where its run begins, so joining needs no search.
#pragma once

#include "../common/util.cuh"

namespace eb {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxEntries = 1024;   // entries that fit a CTA's shared table

struct Prefix {
  int cum[kMaxEntries + 1];         // units of the entries before
  int limit[kMaxEntries];           // keys
};

struct Args {
  const void* q;          // [batch, tokens, heads, dim], dense
  const void* k;          // [pages, kv_heads, page, dim], dense
  const void* v;
  const int* tables;      // [batch, width]
  const int* positions;   // [batch, tokens], -1: no row
  void* out;              // like q
  float* part_o;          // [2 * CTAs, row_tile, dim] partial sums of 2^(a - m) v
  float* part_ml;         // [2 * CTAs, row_tile, 2]: m (base 2), sum of 2^(a - m)
  int* cuts;              // [CTAs, 4]: entry, head, first tile and tiles of the item that a CTA's run begins in
  int* run;               // [1] units of a run
  int batch, tokens, heads, kv_heads, dim;
  int group;              // query heads of an item
  int item_heads;         // items of an entry: kv_heads, or a multiple when an item takes part of a head's group
  int head_div;           // item_heads / kv_heads
  int pages, page, page_shift, width;
  int row_tile;           // rows of a row tile (a whole number of tokens)
  int tile_tokens;        // its tokens
  int row_tiles;          // row tiles of a sequence
  int key_tile;           // keys of a tile
  int flat;               // 1: equal runs of the tile list; 0: one item a CTA (too many entries for the table)
  int item_cost;          // what starting and finishing an item costs, in tiles of work
  int vectors;            // rows and pools allow loads of four elements (general kernel)
  float scale_log2;       // log2(e) / sqrt(dim)
};

struct Segment {
  int entry, head;        // the item
  int batch, token0;      // its sequence and first token
  int begin, end;         // key tiles
  int limit;              // keys of the item
  int slot;               // partial slot, -1: the whole item (written out)
};

// Largest position of an entry's rows plus one, inside the table; 0 when it has no row.
EB_DEVICE int entry_limit(const Args& p, int entry) {
  const int b = entry / p.row_tiles, t0 = (entry - b * p.row_tiles) * p.tile_tokens;
  const int n = min(p.tile_tokens, p.tokens - t0);
  const int* pos = p.positions + static_cast<int64_t>(b) * p.tokens + t0;
  int top = -1;
#pragma unroll 4
  for (int i = 0; i < n; ++i) top = max(top, pos[i]);
  return static_cast<int>(min(static_cast<int64_t>(top) + 1, static_cast<int64_t>(p.width) * p.page));
}

EB_DEVICE int entry_limit_warp(const Args& p, int entry, int lane) {
  const int b = entry / p.row_tiles, t0 = (entry - b * p.row_tiles) * p.tile_tokens;
  const int n = min(p.tile_tokens, p.tokens - t0);
  const int* pos = p.positions + static_cast<int64_t>(b) * p.tokens + t0;
  int top = -1;
  for (int i = lane; i < n; i += 32) top = max(top, pos[i]);
  top = __reduce_max_sync(0xffffffffu, top);
  return static_cast<int>(min(static_cast<int64_t>(top) + 1, static_cast<int64_t>(p.width) * p.page));
}

// Units of an item of `limit` keys: its tiles, then its fixed cost.
EB_DEVICE int entry_units(const Args& p, int limit) { return limit > 0 ? cdiv(limit, p.key_tile) + p.item_cost : 0; }

// Limits of the entries and prefix of their units; all threads.
EB_DEVICE void build_prefix(const Args& p, Prefix& table) {
  const int entries = p.batch * p.row_tiles;
  int* cum = table.cum;
  if (p.tile_tokens <= 16) {
    for (int e = threadIdx.x; e < entries; e += blockDim.x) {
      const int n = entry_limit(p, e);
      table.limit[e] = n;
      cum[e + 1] = entry_units(p, n);
    }
  } else {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int e = warp; e < entries; e += blockDim.x >> 5) {
      const int n = entry_limit_warp(p, e, lane);
      if (lane == 0) {
        table.limit[e] = n;
        cum[e + 1] = entry_units(p, n);
      }
    }
  }
  if (threadIdx.x == 0) cum[0] = 0;
  __syncthreads();
  if (threadIdx.x < 32) {
    int carry = 0;
    for (int base = 0; base < entries; base += 32) {
      const int i = base + threadIdx.x;
      int x = i < entries ? cum[i + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (static_cast<int>(threadIdx.x) >= o) x += y;
      }
      x += carry;
      if (i < entries) cum[i + 1] = x;
      carry = __shfl_sync(0xffffffffu, x, 31);
    }
  }
  __syncthreads();
}

// Units of one run (all of a call's units fit an int: see the launch).
EB_DEVICE int run_units(const Args& p, int total, int ctas) {
  const int all = total * p.item_heads;
  return all / ctas + (all % ctas != 0);
}

// Walks the segments of one CTA's run. `table` is unused when flat == 0.
struct Walk {
  int at, end, first;
  int entry_hint;

  EB_DEVICE void start(const Args& p, const Prefix& table) {
    if (p.flat) {
      const int* cum = table.cum;
      const int total = cum[p.batch * p.row_tiles];
      const int run = run_units(p, total, gridDim.x), all = total * p.item_heads;
      at = static_cast<int>(min(static_cast<int64_t>(blockIdx.x) * run, static_cast<int64_t>(all)));
      end = all - at < run ? all : at + run;
    } else {
      // Latest row tiles first: they hold the most keys of a causal chunk.
      at = p.batch * p.row_tiles * p.item_heads - 1 - static_cast<int>(blockIdx.x);
      end = at + 1;
    }
    first = at;
    entry_hint = 0;
  }

  // The next segment, or false. Uniform over the threads that call it. In the
  // one-item form the segment may be empty (begin == end, slot -1): the output is zero.
  EB_DEVICE bool next(const Args& p, const Prefix& table, Segment& s) {
    const int* cum = table.cum;
    while (true) {
      if (at >= end) return false;
      const int here = at;
      if (!p.flat) {
        s.entry = at / p.item_heads;
        s.head = at - s.entry * p.item_heads;
        s.slot = -1;
        ++at;
      } else {
        const int entries = p.batch * p.row_tiles;
        int lo = entry_hint, hi = entries;
        while (hi - lo > 1) {   // last entry whose items start at or before `at` (never an empty one)
          const int mid = (lo + hi) >> 1;
          if (cum[mid] * p.item_heads <= at) lo = mid;
          else hi = mid;
        }
        s.entry = lo;
        entry_hint = lo;
        const int units = cum[lo + 1] - cum[lo], tiles = units - p.item_cost;
        const int rel = at - cum[lo] * p.item_heads;
        s.head = rel / units;
        const int unit = rel - s.head * units;
        const int n = min(units - unit, end - at);
        s.begin = min(unit, tiles);
        s.end = min(unit + n, tiles);
        at += n;
        if (s.begin == s.end) continue;   // only the item's fixed cost fell into this run
        s.slot = s.begin == 0 && s.end == tiles ? -1 : 2 * static_cast<int>(blockIdx.x) + (here == first ? 0 : 1);
      }
      s.batch = s.entry / p.row_tiles;
      s.token0 = (s.entry - s.batch * p.row_tiles) * p.tile_tokens;
      return true;
    }
  }
};

// What the combine kernel needs, and the rows of entries without any key. All threads, after walk.start().
template <typename T>
EB_DEVICE void publish_run(const Args& p, const Prefix& table, const Walk& walk) {
  if (!p.flat) return;
  const int* cum = table.cum;
  if (threadIdx.x == 0) {
    Walk probe = walk;
    Segment s;
    int4 cut = make_int4(0, 0, 0, 0);
    if (probe.next(p, table, s)) cut = make_int4(s.entry, s.head, s.begin, cum[s.entry + 1] - cum[s.entry] - p.item_cost);
    reinterpret_cast<int4*>(p.cuts)[blockIdx.x] = cut;
    if (blockIdx.x == 0) *p.run = run_units(p, cum[p.batch * p.row_tiles], gridDim.x);
  }
  // Every CTA takes a share of each such entry: the last tiles of a ragged batch may all be empty.
  const int entries = p.batch * p.row_tiles;
  const int64_t row = static_cast<int64_t>(p.heads) * p.dim * sizeof(T);
  const int64_t at = blockIdx.x * blockDim.x + threadIdx.x, step = gridDim.x * blockDim.x;
  for (int e = 0; e < entries; ++e) {
    if (cum[e + 1] != cum[e]) continue;
    const int b = e / p.row_tiles, t0 = (e - b * p.row_tiles) * p.tile_tokens;
    const int64_t n = min(p.tile_tokens, p.tokens - t0) * row;
    char* out = static_cast<char*>(p.out) + (static_cast<int64_t>(b) * p.tokens + t0) * row;
    if (row % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0) {
      for (int64_t i = at * 16; i < n; i += step * 16) *reinterpret_cast<uint4*>(out + i) = make_uint4(0, 0, 0, 0);
    } else {   // an even number of elements of two bytes or more
      for (int64_t i = at * 4; i < n; i += step * 4) *reinterpret_cast<uint32_t*>(out + i) = 0;
    }
  }
}

// Limit of a segment's item, and for the one-item form its tiles; every thread of a warp calls it.
EB_DEVICE void finish_segment(const Args& p, const Prefix& table, Segment& s, int lane) {
  if (p.flat) {
    s.limit = table.limit[s.entry];
  } else {
    s.limit = entry_limit_warp(p, s.entry, lane);
    s.begin = 0;
    s.end = cdiv(s.limit, p.key_tile);
  }
}

}  // namespace paged

// Joins the partial sums of cut items (paged_combine.cu).
template <typename T>
void paged_combine_launch(const paged::Args& args, int ctas, cudaStream_t stream);

}  // namespace eb
