// Attention over shared prefixes: what the kernels are told, and how the work is divided.
//
// Request b has the rows cu[b] .. cu[b + 1] - 1 of q (one row, its own number, without cu); the i-th of n sees the
// prefix of the request's group and the request's own tokens 0 .. length - n + i.  Whatever the tables, lengths and
// starts hold, nothing outside q, the cache, the scratch and the result is touched: lengths are cut to their tables, rows to
// q, and an entry that is no page of the cache is taken for the nearest.
//
// A kernel's row is a (token, query head) pair; the query heads of a kv head are in `chunks` chunks of up to `heads`, and a
// tile of rows is `tokens` tokens of a chunk.  Keys come in tiles, too.  Two kinds of work leave pieces of results, each a
// maximum (in log2 units), a sum and the weighted values of every row:
//  * a group's prefix (PrefixItem): the group's rows in tiles, its keys in chunks of `chunk` tiles, the same for all groups;
//    every item's piece has a place of its own.  Row tiles of one chunk of keys are neighbours, so that they read it at the
//    same time.
//  * a request's own tokens (Cursor): the tiles of all requests (and of their tiles of rows) are one long sequence, and
//    every warp takes an equal run of it, so that warps end together whatever the lengths.  A run begins and ends inside
//    requests; what is cut has the warp's two places, the rest a row's own.
// The joining kernel works the same arithmetic out again and adds a row's pieces up, in order: no atomics.
#pragma once
#include "common.cuh"

namespace gf {

struct PrefixArgs {
  const void* q;
  const void* k;               // pages [pages][page][nkv][hd]
  const void* v;
  const int* prefix_table;     // [G][prefix_stride]
  const int* prefix_lens;      // [G]
  const int* table;            // [B][table_stride]
  const int* lengths;          // [B]
  const int* cu_groups;        // [G + 1], or null: all requests are of group 0
  const int* cu;               // [B + 1], or null: a row a request
  void* out;                   // [T][nh][hd]
  int q_stride, prefix_stride, table_stride, prefix_limit, limit, G, B, T, nh, nkv, page, pages, page_shift;
  float scale;
};

// ------------------------------------------------------------------------------------- what a call says
struct Rows {
  int first, count;
};
__device__ __forceinline__ int row_start(const PrefixArgs& a, int b) {
  return a.cu ? min(max(fresh_index(a.cu + b), 0), a.T) : min(b, a.T);
}
__device__ __forceinline__ Rows rows_of(const PrefixArgs& a, int b) {
  const int first = row_start(a, b);
  return {first, max((a.cu ? row_start(a, b + 1) : min(b + 1, a.T)) - first, 0)};
}
__device__ __forceinline__ int own_length(const PrefixArgs& a, int b) {
  return min(max(fresh_index(a.lengths + b), 0), a.limit);
}
__device__ __forceinline__ int prefix_length(const PrefixArgs& a, int g) {
  return g < 0 ? 0 : min(max(fresh_index(a.prefix_lens + g), 0), a.prefix_limit);
}
// A request's group; -1: none, it has no prefix.
__device__ __forceinline__ int group_of(const PrefixArgs& a, int b) {
  if (!a.cu_groups) return a.G > 0 ? 0 : -1;
  int low = 0, high = a.G;                 // the first g whose end is behind b
  while (low < high) {
    const int mid = (low + high) >> 1;
    if (fresh_index(a.cu_groups + mid + 1) > b) high = mid;
    else low = mid + 1;
  }
  return low < a.G && fresh_index(a.cu_groups + low) <= b ? low : -1;
}
// The rows of a group's requests.
__device__ __forceinline__ Rows group_rows(const PrefixArgs& a, int g) {
  const int b0 = a.cu_groups ? min(max(fresh_index(a.cu_groups + g), 0), a.B) : 0;
  const int b1 = a.cu_groups ? min(max(fresh_index(a.cu_groups + g + 1), b0), a.B) : a.B;
  const int first = row_start(a, b0);
  return {first, max(row_start(a, b1) - first, 0)};
}
__device__ __forceinline__ int page_in(const PrefixArgs& a, int number) {
  return min(max(number, 0), a.pages - 1);
}
__device__ __forceinline__ int logical_page(const PrefixArgs& a, int c) {
  return a.page_shift >= 0 ? c >> a.page_shift : c / a.page;
}
// The place of token c of the sequence that a row of a table names.
__device__ __forceinline__ int slot_of(const PrefixArgs& a, const int* tbl, int c) {
  const int lp = logical_page(a, c);
  return page_in(a, fresh_index(tbl + lp)) * a.page + (c - lp * a.page);
}

// a / b for numbers that are small as a rule (a 64-bit division takes longer than the rest of the division of the work).
__device__ __forceinline__ long long quotient(long long a, long long b) {
  return (a | b) >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b);
}

// ------------------------------------------------------------------------------------- rows
struct Shape {
  int chunks, heads, tokens;    // chunks of a kv head's query heads, heads of a chunk at most, tokens of a row tile
};
__host__ __device__ __forceinline__ Shape row_shape_of(int nh, int nkv, int rows) {
  const int each = nh / nkv, chunks = (each + rows - 1) / rows, heads = (each + chunks - 1) / chunks;
  return {chunks, heads, rows / heads};
}

// ------------------------------------------------------------------------------------- prefixes
struct PrefixItem {
  int g, hc, split, m;          // hc: kv head * chunks + chunk; m: the tile of rows
  int first, count;             // its tokens
  int length, tiles;            // of the prefix
};
// Groups' numbers of row tiles and key tiles, a lane a group of 32.
struct GroupTiles {
  int mt, nt, first, count, length;
  __device__ __forceinline__ void load(const PrefixArgs& a, int g, int tokens, int tile) {
    mt = nt = first = count = length = 0;
    if (g < a.G) {
      const Rows r = group_rows(a, g);
      first = r.first, count = r.count;
      length = prefix_length(a, g);
      mt = (count + tokens - 1) / tokens;
      nt = (length + tile - 1) / tile;
    }
  }
};
// The prefixes' work, by one warp: row tiles times key tiles of all heads, the same with what starts and ends cost, and the longest
// prefix.  `t` keeps the first 32 groups.
// Tiles that an item costs beside its own.  (Without it few key tiles of many rows had too few SMs: 252 requests of up to 5 rows behind
// 74 tokens, 40 heads on 8 of 128, 496 us, 199 at 3, 196 at 6; 64 of one row behind 400, 28 on 4, 42.6, 40.9, 31.8.)
constexpr int kFarOver = 6;
struct FarWork {
  long long units, priced;
  int most;
};
__device__ __forceinline__ FarWork far_work(const PrefixArgs& a, GroupTiles& t, int H, int tokens, int tile) {
  const int lane = threadIdx.x & 31;
  t.load(a, lane, tokens, tile);
  FarWork w{(long long)t.mt * H * t.nt, t.nt ? (long long)t.mt * H * (t.nt + kFarOver) : 0, t.mt ? t.nt : 0};
  for (int g0 = 32; g0 < a.G; g0 += 32) {
    GroupTiles u;
    u.load(a, g0 + lane, tokens, tile);
    w.units += (long long)u.mt * H * u.nt;
    w.priced += u.nt ? (long long)u.mt * H * (u.nt + kFarOver) : 0;
    w.most = max(w.most, u.mt ? u.nt : 0);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    w.units += __shfl_xor_sync(0xffffffffu, w.units, o);
    w.priced += __shfl_xor_sync(0xffffffffu, w.priced, o);
    w.most = max(w.most, __shfl_xor_sync(0xffffffffu, w.most, o));
  }
  return w;
}
// A row's pieces are read one after the other when they are joined: no prefix is cut into more chunks than this.
constexpr int kMostSplits = 24, kMostSplitsOfWarps = 64;      // (by blocks, by single warps)
// Tiles of a chunk of keys, by one warp.  With `workers` blocks the time is about (rounds of items) * (chunk + over),
// over: what an item's start and end cost in tiles.  Looked at are the 32 lengths from one, a half and a third of an equal share
// on; the longest prefix, which is always possible, is the last resort.
__device__ __forceinline__ int plan_chunk(const PrefixArgs& a, const GroupTiles& first, const FarWork& all, int H, int tokens, int tile,
                                          int workers, int places, int over, int most_splits = kMostSplits) {
  const int lane = threadIdx.x & 31;
  if (all.most == 0) return 1;
  GroupTiles t = first;
  int len[3];
  int items[3] = {0, 0, 0};
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const long long share = quotient(all.units + (long long)workers * (k + 1) - 1, (long long)workers * (k + 1));
    const int from = max((int)(share < all.most ? share : all.most), (all.most + most_splits - 1) / most_splits);
    len[k] = min(all.most, max(1, from) + lane * max(1, from / 48));
  }
  if (lane == 31) len[0] = all.most;
  for (int g0 = 0; g0 < a.G; g0 += 32) {
    if (g0) t.load(a, g0 + lane, tokens, tile);
    for (int i = 0; i < min(32, a.G - g0); ++i) {
      const int mt = __shfl_sync(0xffffffffu, t.mt, i) * H, nt = __shfl_sync(0xffffffffu, t.nt, i);
#pragma unroll
      for (int k = 0; k < 3; ++k) items[k] += mt * ((nt + len[k] - 1) / len[k]);
    }
  }
  float best = INFINITY;
  int chunk = all.most;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const float rounds = (float)((items[k] + workers - 1) / workers), cost = rounds * (len[k] + over);
    if (items[k] <= places && (cost < best || (cost == best && len[k] > chunk))) best = cost, chunk = len[k];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float other = __shfl_xor_sync(0xffffffffu, best, o);
    const int c = __shfl_xor_sync(0xffffffffu, chunk, o);
    if (other < best || (other == best && c > chunk)) best = other, chunk = c;
  }
  return chunk;
}
// What the joining kernel needs of a group: its first item, its prefix's chunks, its tiles of rows and its first row.
struct FarPlan {
  int base, splits, mt, first;
};
// By one warp; `t` has the first 32 groups.
__device__ __forceinline__ void write_far_plan(const PrefixArgs& a, const GroupTiles& first, int H, int tokens, int tile, int chunk,
                                               FarPlan* plan) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  GroupTiles t = first;
  for (int g0 = 0; g0 < a.G; g0 += 32) {
    if (g0) t.load(a, g0 + lane, tokens, tile);
    const int splits = (t.nt + chunk - 1) / chunk, items = t.mt * H * splits;
    int sum = items;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (g0 + lane < a.G) plan[g0 + lane] = {before + sum - items, splits, t.mt, t.first};
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
}
// Item `index` in the order groups, (kv head, chunk of heads), chunks of keys, tiles of rows; false behind the last.
// By a whole warp; `t` keeps the first 32 groups' tiles.
__device__ __forceinline__ bool find_item(const PrefixArgs& a, const GroupTiles& t, int H, int tokens, int tile, int chunk,
                                          int index, PrefixItem& it) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int g0 = 0; g0 < a.G; g0 += 32) {
    GroupTiles mine = t;
    if (g0) mine.load(a, g0 + lane, tokens, tile);
    const int splits = (mine.nt + chunk - 1) / chunk, items = mine.mt * H * splits;
    int sum = items;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const unsigned has = __ballot_sync(0xffffffffu, index < before + sum);
    if (has) {
      const int who = __ffs(has) - 1;
      const int mt = __shfl_sync(0xffffffffu, mine.mt, who), s = __shfl_sync(0xffffffffu, splits, who);
      const int rest = index - before - __shfl_sync(0xffffffffu, sum - items, who);
      it.g = g0 + who;
      it.m = rest % mt;
      it.split = rest / mt % s;
      it.hc = rest / mt / s;
      const int all = __shfl_sync(0xffffffffu, mine.count, who);
      it.first = __shfl_sync(0xffffffffu, mine.first, who) + it.m * tokens;
      it.count = min(tokens, all - it.m * tokens);
      it.length = __shfl_sync(0xffffffffu, mine.length, who);
      it.tiles = __shfl_sync(0xffffffffu, mine.nt, who);
      return true;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}

// ------------------------------------------------------------------------------------- requests' own tokens
// What a request's start and end cost beside its tiles, in tiles: waiting for its numbers, its rows of q, joining the warps.
constexpr int kItemTiles = 4;
struct Request {
  int first, count, len, shared, g;     // its rows, its own tokens, tokens of the prefix (0 where that is another kernel's)
  int far, near;                        // tiles of the prefix, of the own tokens
  __device__ __forceinline__ int tiles() const { return max(1, far + near); }
  __device__ __forceinline__ int units() const { return tiles() + kItemTiles; }
  __device__ __forceinline__ int row_tiles(int tokens) const { return (count + tokens - 1) / tokens; }
};
__device__ __forceinline__ Request request_of(const PrefixArgs& a, int b, bool both, int tile) {
  Request r;
  r.g = -1, r.shared = 0;
  if (both && a.G == 1) {
    // (one group: nothing waits for anything)
    const int length = prefix_length(a, 0);
    const bool in = !a.cu_groups || (fresh_index(a.cu_groups) <= b && b < fresh_index(a.cu_groups + 1));
    r.g = in ? 0 : -1, r.shared = in ? length : 0;
  }
  const Rows rows = rows_of(a, b);
  r.first = rows.first, r.count = rows.count, r.len = own_length(a, b);
  if (both && a.G > 1) r.g = group_of(a, b), r.shared = prefix_length(a, r.g);
  r.far = (r.shared + tile - 1) / tile, r.near = (r.len + tile - 1) / tile;
  return r;
}
// Where a warp's run is: units `off` on of the row tile `rt` of request b, for heads hc.
struct Cursor {
  int hc, b, rt, off;
  long long todo;
  Request req;
};
// What the joining kernel needs of the division: a run's units, the units of one (kv head, chunk of heads), and of every request
// the units before it, its rows, its tiles and its group.
struct OwnPlan {
  long long run, each;
  struct Entry {
    long long base;
    int first, count, tiles, g;
  } of[1];                      // [B]
};
constexpr int kLeastRun = 8;    // the fewest units of a run

// The units of the requests of a block's first THREADS threads, a neighbouring share of all requests each, and of all before and
// in all.
struct OwnWork {
  int b0, b1;
  long long mine, start, total;
  Request first;                // b0's
  __device__ __forceinline__ Request request(const PrefixArgs& a, int b, bool both, int tile) const {
    return b == b0 ? first : request_of(a, b, both, tile);
  }
};
template <int THREADS>
__device__ __forceinline__ OwnWork own_work(const PrefixArgs& a, int tokens, int tile, bool both, long long* counts) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, each = (a.B + THREADS - 1) / THREADS;
  OwnWork w{min((int)threadIdx.x * each, a.B), 0, 0, 0, 0, {}};
  w.b1 = min(w.b0 + each, a.B);
  if (threadIdx.x < THREADS)
    for (int b = w.b0; b < w.b1; ++b) {
      const Request r = request_of(a, b, both, tile);
      if (b == w.b0) w.first = r;
      w.mine += (long long)r.row_tiles(tokens) * r.units();
    }
  long long sum = w.mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  if (lane == 31 && warp < THREADS / 32) counts[warp] = sum;
  __syncthreads();
  w.start = sum - w.mine;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) {
    if (i < warp) w.start += counts[i];
    w.total += counts[i];
  }
  return w;
}
// What the threads that counted leave for the warps' searches.
template <int THREADS> struct OwnShares {
  long long start[THREADS + 1];
  Request first[THREADS];
};
// The run of warp `me` of `runs` of them, by that warp; all threads of the block call.  `plan`: where the division is written down, by
// the block that is given it.
template <int THREADS>
__device__ __forceinline__ Cursor find_run(const PrefixArgs& a, const OwnWork& w, OwnShares<THREADS>& shares, int H, int tokens,
                                           int tile, bool both, long long me, long long runs, OwnPlan* plan) {
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < THREADS) {
    shares.start[threadIdx.x] = w.start, shares.first[threadIdx.x] = w.first;
    if (threadIdx.x == 0) shares.start[THREADS] = w.total;
  }
  __syncthreads();
  const long long all = w.total * H, share = quotient(all + runs - 1, runs);
  const long long run = share > kLeastRun ? share : kLeastRun, at = run * me;
  if (plan && threadIdx.x < THREADS) {
    if (threadIdx.x == 0) plan->run = run, plan->each = w.total;
    long long base = w.start;
    for (int b = w.b0; b < w.b1; ++b) {
      const Request r = w.request(a, b, both, tile);
      plan->of[b] = {base, r.first, r.count, r.tiles(), both ? r.g : group_of(a, b)};
      base += (long long)r.row_tiles(tokens) * r.units();
    }
  }
  Cursor c{};
  if (me >= runs || at >= all) return c;
  c.hc = (int)quotient(at, w.total);
  long long rest = at - c.hc * w.total;
  // the thread that counted the request
  int who = 0;
#pragma unroll
  for (int j = 0; j < THREADS / 32; ++j) {
    const unsigned hit = __ballot_sync(0xffffffffu, shares.start[32 * j + lane] <= rest && rest < shares.start[32 * j + lane + 1]);
    if (hit) who = 32 * j + __ffs(hit) - 1;
  }
  rest -= shares.start[who];
  const int each = (a.B + THREADS - 1) / THREADS;
  c.b = who * each, c.req = shares.first[who];
  for (;;) {
    const long long units = c.req.units(), here = c.req.row_tiles(tokens) * units;
    if (rest < here || c.b + 1 >= a.B) {
      c.rt = (int)quotient(rest, units), c.off = (int)(rest - c.rt * units);
      break;
    }
    rest -= here;
    c.req = request_of(a, ++c.b, both, tile);
  }
  c.todo = min(run, all - at);
  return c;
}

// Prefixes and own tokens are worked on side by side, by two launches: of `sms` SMs this many have the prefixes.  A tile of a
// prefix costs `far_cost` of what a tile of own tokens does.
__device__ __forceinline__ int far_share(int sms, long long far_units, float far_cost, long long own_units) {
  if (far_units == 0) return 0;
  const float far = (float)far_units * far_cost, own = (float)own_units;
  const int share = (int)(sms * far / (far + own) + 0.5f);
  return min(max(share, 1), own_units > 0 ? sms - 1 : sms);
}

}  // namespace gf
