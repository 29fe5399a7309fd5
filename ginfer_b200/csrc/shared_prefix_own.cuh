// Requests' own tokens (with their prefixes where nobody else reads those), and in 32 bits the groups' prefixes, too, on mma.sync, a
// warp by itself: few rows, many keys that are read once (see shared_prefix.cuh for how the work is divided).
//
// S^T = K q^T and O^T = V^T P^T: keys, then channels, are the instruction's 16 rows and up to 8 rows of q its columns, NG times.
// A warp has a ring of its own, fills it itself and waits for nobody, so that whatever one of them waits for (a request's
// numbers, its pages, its rows of q) the others' copies are under way.  A tile within its sequence comes by TMA where that
// serves the pages, a box of a page and 64 channels; the last of a sequence comes by cp.async, which leaves zeros behind its
// end: what lies there may be anything.
//
// What bounds it is latency: a request's numbers, its run, its pages and its q come one after the other (about 10 us from the start to
// the first product), then a tile costs a warp 0.8 us.  Own tokens of 64 requests of up to 1,024, 28 heads on 4 of 128, 72 MB, on
// all SMs 28 us, 2.6 TB/s; in 32 bits 12 requests of up to 600 behind up to 2,000, 14 on 2 of 64, as clusters of two blocks 27 us, prefixes among
// them.  Rings a warp of its own and equal runs replaced blocks that share a tile (the call 52 -> 41 us).
//
// In 32 bits both factors of a product are the sum of two tf32 numbers, 22 bits, and a product three of theirs (what is left out
// is 2^-22 of it).  The instruction cuts its sums off instead of rounding them: it adds eight products up from zero, the long
// sums are additions of their own.  (Left to the instruction, results were off by three times as much, heads of 256 by eight times.)
#pragma once
#include "shared_prefix.cuh"

namespace gf {
namespace {
namespace own {

// A tile of KEYS keys in shared memory, keys, then values.  bfloat16: head sizes that are a multiple of 64 as TMA's 128-byte swizzle
// leaves them (64 channels of the keys, then the next 64), others in rows of an odd number of 16-byte chunks.  32 bits: rows 4
// (keys) and 8 (values) banks apart, so that a warp's reads of 8 keys and 4 channels, or of 4 keys and 8 channels, meet every bank once.
template <typename T> struct Tile;
template <> struct Tile<bf16> {
  static constexpr int KEYS = HD <= 64 ? 32 : 16, WARPS = HD <= 128 ? 8 : 4, STAGES = 3;
  static constexpr bool SWIZZLED = HD % 64 == 0;
  static constexpr int HALVES = SWIZZLED ? HD / 64 : 1, PADDED = HD + 8, CHUNK = 8;
  static constexpr uint32_t PLANE = SWIZZLED ? KEYS * HD * 2 : (KEYS * PADDED * 2 + 127) / 128 * 128, STAGE = 2 * PLANE;
  static __device__ __forceinline__ uint32_t place(int plane, int key, int ch) {       // byte offset of CHUNK channels of a key
    if constexpr (SWIZZLED)
      return plane * PLANE + (uint32_t)(ch >> 6) * (KEYS * 128) + (uint32_t)key * 128u + (uint32_t)((((ch >> 3) & 7) ^ (key & 7)) << 4);
    else
      return plane * PLANE + (uint32_t)key * (PADDED * 2) + (uint32_t)ch * 2u;
  }
};
template <> struct Tile<float> {
  static constexpr int KEYS = 16, WARPS = HD <= 64 ? 8 : HD <= 128 ? 4 : 2, STAGES = 3;
  static constexpr bool SWIZZLED = false;
  static constexpr int HALVES = 1, CHUNK = 4;
  static constexpr uint32_t PLANE = KEYS * (HD + 4) * 4, STAGE = PLANE + KEYS * (HD + 8) * 4;
  static __device__ __forceinline__ uint32_t place(int plane, int key, int ch) {
    return plane * PLANE + (uint32_t)(key * (HD + 4 + 4 * plane) + ch) * 4u;
  }
};
constexpr int KCH = HD / 16;
// (joining warps inside a block takes the ring's memory, and what it has not)
template <typename T> __host__ __device__ constexpr uint32_t smem_bytes(int ng) {
  using G = Tile<T>;
  const uint32_t ring = G::WARPS * G::STAGES * G::STAGE, exchange = (G::WARPS + 1) * 8 * ng * (HD + 2) * 4;
  return (ring > exchange ? ring : exchange) + G::WARPS * G::STAGES * 8 + 1024;
}
constexpr float kGrowth = 8.f;   // log2 units: weights stay below 2^8
// Groups of 8 rows at most, of own tokens and of prefixes (in 32 bits): their results and their q have to fit the registers, and
// a tile's steps follow one another: 16 rows of q share what a warp reads, more rows are other warps' work, which reads it
// again from L2.  us, 8 rows / 16 rows: 32 requests of up to 5 rows, 12 heads on 2 kv heads of 128 (30 rows) 43.1 / 38.5 (32 rows 50);
// 64 of up to 3, 28 on 4 of 128 (21 rows, which 16 hold no better than 8 do) 67.1 / 74.9; 24 of up to 3, 16 on 4 of 96 (12 rows) 31 / 35.
// 32-bit, 14 on 2 of 64, requests of up to 2 (14 rows): 64 behind 8,000 145 / 176; 12 behind 2,000, a cluster an item, 27.3 / 23.5.
template <typename T> constexpr int kNearGroups = sizeof(T) == 2 ? 2 : 1;
constexpr int kOneGroup = 16;    // rows of a request up to which 8 are a tile
constexpr int kFarGroups = HD <= 64 ? 2 : 0;

struct Args {
  PrefixArgs a;
  int both, tma;               // both: prefixes, too
  int joined;                  // another kernel adds a row's pieces up; else a cluster's warps have an item, and it is written here
  int cluster;                 // blocks of a cluster then (neighbours along x)
  int after;                   // the launch runs beside the one before it, whose results the joining kernel reads, too
  Shape shape;
  int H, rows;                 // kv heads * chunks; rows of a tile
  int sms;
  Shape far_shape;             // of the prefixes' kernel beside this one
  int far_tile, far_H;
  float far_cost;              // what a tile of a prefix costs, in tiles of this kernel
  OwnPlan* plan;
  float* cut_o;                // [warps][2][rows][HD]: pieces of cut items
  float2* cut_ml;
  float* row_o;                // [T][nh][HD]: of whole items, where a prefix is to be joined
  float2* row_ml;
  int* err;
  // prefixes in 32 bits: rows of this kernel's tiles are far_shape's, and own tokens' are
  Shape own_shape;
  int own_H, places;
  FarPlan* far_plan;           // [G]
  float* far_o;                // [places][rows][HD]
  float2* far_ml;
};

// A part of an item: tiles [from, from + count) of its prefix's tiles, then its own tokens'.
struct Piece {
  int first, tokens, hc, from, count, far, far_len, near_len;
  int last;                    // the last own token that the first token sees; the next one sees one more
  const int *far_table, *near_table;
  int to;
  size_t at;                   // CUT, FAR: the place
};
enum { FINAL, ROW, CUT, FAR_PIECE };
struct Keys {
  const int* table;
  int key0, end;
};
__device__ __forceinline__ Keys keys_of(const Piece& x, int tile, int keys) {
  if (tile < x.far) return {x.far_table, tile * keys, x.far_len};
  return {x.near_table, (tile - x.far) * keys, x.near_len};
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

// 32 bits as two tf32 numbers.
struct Split {
  uint32_t hi, lo;
};
__device__ __forceinline__ Split split(float x) {
  Split s;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(s.hi) : "f"(x));
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(s.lo) : "f"(x - __uint_as_float(s.hi)));
  return s;
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// All threads of a cluster's blocks.
__device__ __forceinline__ void cluster_meet() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// What `addr` of this block is in another one of the cluster.
__device__ __forceinline__ uint32_t in_block(uint32_t addr, int rank) {
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  return there;
}

// A TMA copy of what is read once: it leaves L2 first.
__device__ __forceinline__ void copy_once(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
      ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "l"(policy)
      : "memory");
}

template <typename T, int NG, bool FAR>
__global__ void __launch_bounds__(32 * Tile<T>::WARPS, 1)
prefix_own_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const Args p) {
  using G = Tile<T>;
  constexpr int KEYS = G::KEYS, WARPS = G::WARPS, STAGES = G::STAGES, THREADS = 32 * WARPS;
  constexpr int COUNTING = THREADS;
  constexpr uint32_t STAGE = G::STAGE;
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char* base = raw + ((0u - smem_u32(raw)) & 1023u);               // (a swizzle counts from 1 KB)
  __shared__ long long counts[WARPS];
  __shared__ OwnShares<COUNTING> shares;
  __shared__ int far_s, chunk_s;
  __shared__ GroupTiles groups_s[FAR ? 32 : 1];
  const PrefixArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  unsigned char* ring = base + warp * (STAGES * STAGE);
  uint64_t* full = reinterpret_cast<uint64_t*>(base + smem_bytes<T>(NG) - 1024 - WARPS * STAGES * 8) + warp * STAGES;
  if (lane == 0) {
    for (int i = 0; i < STAGES; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&full[i])), "r"(32));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (!p.after) pdl_wait();
  // FAR: behind the wait, since the kernel beside this one reads what was waited for.  Else the joining kernel's blocks may stand
  // by: every block of this one is running by then.
  if (FAR || p.joined) pdl_trigger();
  Cursor cur{};
  Request req{};
  GroupTiles groups{};
  int chunk = 1, index = 0, stride = 0;
  if constexpr (FAR) {
    // how the prefixes and the own tokens share the SMs, and the prefixes' chunks
    FarWork f{};
    if (warp == WARPS - 1) f = far_work(a, groups, p.H, p.shape.tokens, KEYS);
    const OwnWork w = own_work<COUNTING>(a, p.own_shape.tokens, KEYS, false, counts);
    if (warp == WARPS - 1) {
      const int workers = far_share(p.sms, f.priced, p.far_cost, w.total * p.own_H) * WARPS;
      const int c = plan_chunk(a, groups, f, p.H, p.shape.tokens, KEYS, max(workers, 1), p.places, kItemTiles, kMostSplitsOfWarps);
      groups_s[lane] = groups;
      if (lane == 0) {
        chunk_s = c, far_s = workers;
      }
      if (blockIdx.x == 0) write_far_plan(a, groups, p.H, p.shape.tokens, KEYS, c, p.far_plan);
    }
    __syncthreads();
    groups = groups_s[lane], chunk = chunk_s, stride = far_s;
    index = blockIdx.x * WARPS + warp;
    if (index >= stride) index = p.places;
  } else if (p.joined) {
    // this block's warps' runs
    GroupTiles gt{};
    FarWork f{};
    if (p.after && warp == WARPS - 1) f = far_work(a, gt, p.far_H, p.far_shape.tokens, p.far_tile);
    const OwnWork w = own_work<COUNTING>(a, p.shape.tokens, KEYS, p.both, counts);
    if (threadIdx.x == THREADS - 1) far_s = p.after ? far_share(p.sms, f.priced, p.far_cost, w.total * p.H) : 0;
    __syncthreads();
    const int blocks = p.after ? max(p.sms - far_s, 1) : (int)gridDim.x;
    cur = find_run<COUNTING>(a, w, shares, p.H, p.shape.tokens, KEYS, p.both, (long long)blockIdx.x * WARPS + warp,
                             (long long)blocks * WARPS, blockIdx.x == 0 ? p.plan : nullptr);
    req = cur.req;
  } else {
    cur = {(int)blockIdx.z, (int)blockIdx.y, (int)blockIdx.x / p.cluster, 0, 0, {}};
    req = request_of(a, cur.b, p.both, KEYS);
    __syncthreads();
  }
  const int each = a.nh / a.nkv;
  const float scale_log2 = a.scale * LOG2E;
  const int box = min(a.page, KEYS), boxes = KEYS / box;
  const bool tma = G::SWIZZLED && p.tma;
  uint64_t once;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(once));
  uint32_t phases = 0, written = 0;      // a bit a stage; written: by cp.async
  int st = 0;
  bool ok = true;
  // the next piece of this warp's run (or its share of the block's item)
  auto next = [&](Piece& x) {
    auto set = [&](int from, int count) {
      const int done = cur.rt * p.shape.tokens;
      x.first = req.first + done, x.tokens = min(p.shape.tokens, req.count - done), x.hc = cur.hc;
      x.from = from, x.count = count;
      x.far = req.far, x.far_len = req.shared, x.near_len = req.len, x.last = req.len - req.count + done;
      x.far_table = a.prefix_table + (size_t)max(req.g, 0) * a.prefix_stride;
      x.near_table = a.table + (size_t)cur.b * a.table_stride;
    };
    if constexpr (FAR) {
      PrefixItem it;
      if (index >= p.places || !find_item(a, groups, p.H, p.shape.tokens, KEYS, chunk, index, it)) return false;
      x.first = it.first, x.tokens = it.count, x.hc = it.hc;
      x.from = it.split * chunk, x.count = min(chunk, it.tiles - x.from);
      x.far = it.tiles, x.far_len = it.length, x.near_len = 0, x.last = -1;
      x.far_table = a.prefix_table + (size_t)it.g * a.prefix_stride, x.near_table = nullptr;
      x.to = FAR_PIECE, x.at = index;
      index += stride;
      return true;
    }
    if (!p.joined) {
      if (cur.rt * p.shape.tokens >= req.count) return false;
      const int tiles = req.far + req.near, all = WARPS * p.cluster, me = (int)blockIdx.x % p.cluster * WARPS + warp;
      const int w0 = tiles * me / all, w1 = tiles * (me + 1) / all;
      set(w0, w1 - w0);
      x.to = FINAL;
      cur.rt += gridDim.x / p.cluster;
      return true;
    }
    while (cur.todo > 0) {
      const int tiles = req.tiles(), units = req.units(), from = cur.off;
      const int count = (int)min(cur.todo, (long long)(units - from));
      const bool some = from < tiles;              // (else only the item's end, which costs time and has no tiles)
      if (some) {
        set(from, min(count, tiles - from));
        const bool starts = from == 0, ends = from + x.count == tiles;
        x.to = starts && ends ? (p.both ? FINAL : ROW) : CUT;
        x.at = ((size_t)blockIdx.x * WARPS + warp) * 2 + (starts ? 1 : 0);
        if (req.far + req.near == 0) x.count = 0;  // (an item without a key)
      }
      cur.todo -= count, cur.off = 0;
      if (cur.todo > 0 && ++cur.rt >= req.row_tiles(p.shape.tokens)) {
        cur.rt = 0;
        do {
          if (++cur.b == a.B) cur.b = 0, ++cur.hc;
          req = request_of(a, cur.b, p.both, KEYS);
        } while (req.count == 0);
      }
      if (some) return true;
    }
    return false;
  };
  Piece x;
  while (next(x)) {
    const int kvh = x.hc / p.shape.chunks, part = x.hc - kvh * p.shape.chunks;
    const int h0 = kvh * each + part * p.shape.heads, heads = min(p.shape.heads, each - part * p.shape.heads);
    const int rows = x.tokens * heads;
    // ---- copies: a tile's places are looked up one tile ahead
    auto look = [&](int i) {
      const Keys k = keys_of(x, x.from + i, KEYS);
      return slot_of(a, k.table, min(k.key0 + (lane & (KEYS - 1)), k.end - 1));
    };
    auto issue = [&](int i, int slot, int stage_i) {
      const Keys k = keys_of(x, x.from + i, KEYS);
      unsigned char* stage = ring + stage_i * STAGE;
      uint64_t* bar = &full[stage_i];
      if (tma && k.key0 + KEYS <= k.end) {
        // (what this warp's cp.async wrote there is out of the way of the copies)
        if (written >> stage_i & 1) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          written &= ~(1u << stage_i);
        }
        if (lane == 0)
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(STAGE) : "memory");
        else
          asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
        __syncwarp();
        const int bx = lane % boxes, half = lane / boxes % G::HALVES, plane = lane / (boxes * G::HALVES);
        const int row = __shfl_sync(0xffffffffu, slot, bx * box);
        if (plane < 2)
          copy_once(stage + plane * G::PLANE + half * (KEYS * 128) + bx * box * 128, plane ? &vmap : &kmap, bar, kvh * HD + half * 64, row,
                    once);
      } else {
        constexpr int CH = HD / G::CHUNK;
        const T* kp = static_cast<const T*>(a.k) + (size_t)kvh * HD;
        const T* vp = static_cast<const T*>(a.v) + (size_t)kvh * HD;
#pragma unroll 2
        for (int j = 0; j < KEYS * CH / 32; ++j) {
          const int idx = j * 32 + lane, row = idx / CH, ch = (idx - row * CH) * G::CHUNK;
          const size_t off = (size_t)__shfl_sync(0xffffffffu, slot, row) * (a.nkv * HD) + ch;
          const bool there = k.key0 + row < k.end;
          cp_async16(stage + G::place(0, row, ch), kp + off, there);
          cp_async16(stage + G::place(1, row, ch), vp + off, there);
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
        written |= 1u << stage_i;
      }
    };
    int slot = 0;
    if (!ok) x.count = 0;      // (behind a wait that ran out: the warps still meet where they join)
    int first[STAGES];
#pragma unroll
    for (int i = 0; i < STAGES; ++i) first[i] = i < x.count ? look(i) : 0;
    if (STAGES < x.count) slot = look(STAGES);
    // ---- q as the 8-column operand: thread (g, t) has of row 8 ng + g the channels 16 kc + 2t, + 1 and + 8, + 9 (bfloat16), or
    // 8 kc + t and + 4 (32 bits)
    uint32_t qf[NG][sizeof(T) == 2 ? KCH : 2 * KCH][2];
    int see[NG][2];            // the last own token that rows 2t and 2t + 1 see (rows that are none see all, and nobody sees them)
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int r = 8 * n + g, token = r < rows ? r / heads : 0, head = r < rows ? r - token * heads : 0;
      const T* q = static_cast<const T*>(a.q) + (size_t)(x.first + token) * a.q_stride + (size_t)(h0 + head) * HD;
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int kc = 0; kc < KCH; ++kc) {
          qf[n][kc][0] = r < rows ? __ldcg(reinterpret_cast<const unsigned*>(q + 2 * t + kc * 16)) : 0u;
          qf[n][kc][1] = r < rows ? __ldcg(reinterpret_cast<const unsigned*>(q + 2 * t + kc * 16 + 8)) : 0u;
        }
      } else {
#pragma unroll
        for (int kc = 0; kc < 2 * KCH; ++kc) {
          qf[n][kc][0] = r < rows ? __ldcg(reinterpret_cast<const unsigned*>(q + t + kc * 8)) : 0u;
          qf[n][kc][1] = r < rows ? __ldcg(reinterpret_cast<const unsigned*>(q + t + kc * 8 + 4)) : 0u;
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) see[n][e] = 8 * n + 2 * t + e < rows ? x.last + (8 * n + 2 * t + e) / heads : 0x7fffffff;
    }
#pragma unroll
    for (int i = 0; i < STAGES; ++i)
      if (i < x.count) issue(i, first[i], (st + i) % STAGES);
    float o[NG][HD / 16][4], m[NG][2], l[NG][4];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = l[n][2] = l[n][3] = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }
    // ---- tiles
    for (int i = 0; i < x.count && ok; ++i) {
      const Keys k = keys_of(x, x.from + i, KEYS);
      const bool far = x.from + i < x.far;
      // (the warp's verdict: a lane that left by itself would leave the others at the exchanges that follow)
      ok = __all_sync(0xffffffffu, wait_bar(&full[st], (phases >> st) & 1u, p.err, 22));
      if (!ok) break;
      phases ^= 1u << st;
      const unsigned char* stage = ring + st * STAGE;
      // what all rows see needs no comparison: the first token's sight, the sequence's end
      const bool masked = k.key0 + KEYS > k.end || (!far && k.key0 + KEYS - 1 > x.last);
#pragma unroll
      for (int sub = 0; sub < KEYS / 16; ++sub) {
        float s[NG][4];
#pragma unroll
        for (int n = 0; n < NG; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
        if constexpr (sizeof(T) == 2) {
          // (few groups: two sums of every other 16 channels, half as long a chain of products)
          constexpr int SUMS = NG <= 2 && KCH > 1 ? 2 : 1;
          float part[NG][4] = {};
#pragma unroll
          for (int kc = 0; kc < KCH; ++kc) {
            uint32_t af[4];
            ldsm_x4(af, stage + G::place(0, sub * 16 + (lane & 15), kc * 16 + (lane >> 4) * 8));
#pragma unroll
            for (int n = 0; n < NG; ++n) mma16816(kc % SUMS ? part[n] : s[n], af, qf[n][kc][0], qf[n][kc][1]);
          }
          if constexpr (SUMS == 2) {
#pragma unroll
            for (int n = 0; n < NG; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) s[n][i] += part[n][i];
          }
        } else {
#pragma unroll
          for (int kc = 0; kc < 2 * KCH; ++kc) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const Split y = split(*reinterpret_cast<const float*>(stage + G::place(0, g + 8 * (i & 1), kc * 8 + t + 4 * (i >> 1))));
              hi[i] = y.hi, lo[i] = y.lo;
            }
#pragma unroll
            for (int n = 0; n < NG; ++n) {
              const Split q0 = split(__uint_as_float(qf[n][kc][0])), q1 = split(__uint_as_float(qf[n][kc][1]));
              float y[4] = {};
              mma_tf32(y, lo, q0.hi, q1.hi);
              mma_tf32(y, hi, q0.lo, q1.lo);
              mma_tf32(y, hi, q0.hi, q1.hi);
#pragma unroll
              for (int i = 0; i < 4; ++i) s[n][i] += y[i];
            }
          }
        }
        uint32_t b0[NG], b1[NG];           // bfloat16: weights as the 8-column operand
        float w[NG][4];                    // 32 bits: weights as they are
        // what weights are relative to follows a row's largest score only when that has outgrown it by 2^kGrowth: as a rule a
        // tile needs no exchange between lanes
        bool grew = false;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const int ka = k.key0 + sub * 16 + g, kb = ka + 8;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[n][e] *= scale_log2, s[n][2 + e] *= scale_log2;
            if (masked) {
              const int end = far ? k.end - 1 : min(see[n][e], k.end - 1);
              if (ka > end) s[n][e] = -INFINITY;
              if (kb > end) s[n][2 + e] = -INFINITY;
            }
            grew |= fmaxf(s[n][e], s[n][2 + e]) > m[n][e] + kGrowth;
          }
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float top = fmaxf(s[n][e], s[n][2 + e]);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
              if (!(top > m[n][e] + kGrowth)) continue;
              const float corr = fast_exp2(m[n][e] - top);                       // (0 for the first)
              m[n][e] = top, l[n][e] *= corr;
#pragma unroll
              for (int c = 0; c < HD / 16; ++c) o[n][c][e] *= corr, o[n][c][2 + e] *= corr;
            }
          __syncwarp();              // (the matrix instructions want the warp as one)
        }
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          // (-inf - -inf is no number)
          const float base0 = m[n][0] == -INFINITY ? 0.f : m[n][0], base1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
          const float p0 = fast_exp2(s[n][0] - base0), p1 = fast_exp2(s[n][1] - base1);
          const float p2 = fast_exp2(s[n][2] - base0), p3 = fast_exp2(s[n][3] - base1);
          // (weights are rounded to bfloat16 for the product, as everywhere in this package; what is summed are the rounded ones,
          // by a product with ones: a row that one key takes nearly all of gets its value as it is)
          if constexpr (sizeof(T) == 2) {
            const uint32_t ones[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
            b0[n] = transposed(pack_bf16(p0, p1));
            b1[n] = transposed(pack_bf16(p2, p3));
            mma16816(l[n], ones, b0[n], b1[n]);
          } else {
            l[n][0] += p0 + p2;
            l[n][1] += p1 + p3;
            w[n][0] = p0, w[n][1] = p1, w[n][2] = p2, w[n][3] = p3;
          }
        }
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int c = 0; c < HD / 16; ++c) {
            uint32_t af[4];
            ldsm_x4_t(af, stage + G::place(1, sub * 16 + (lane >> 4) * 8 + (lane & 7), c * 16 + ((lane >> 3) & 1) * 8));
#pragma unroll
            for (int n = 0; n < NG; ++n) mma16816(o[n][c], af, b0[n], b1[n]);
          }
        } else {
#pragma unroll
          for (int half = 0; half < 2; ++half) {     // eight keys each
            // the weight of key t (and t + 4) for row g: thread (key, row / 2) has it
            Split p0[NG], p1[NG];
#pragma unroll
            for (int n = 0; n < NG; ++n) {
              const float e0 = __shfl_sync(0xffffffffu, w[n][2 * half], t * 4 + (g >> 1)), e1 = __shfl_sync(0xffffffffu, w[n][2 * half + 1], t * 4 + (g >> 1));
              const float f0 = __shfl_sync(0xffffffffu, w[n][2 * half], (t + 4) * 4 + (g >> 1));
              const float f1 = __shfl_sync(0xffffffffu, w[n][2 * half + 1], (t + 4) * 4 + (g >> 1));
              p0[n] = split(g & 1 ? e1 : e0), p1[n] = split(g & 1 ? f1 : f0);
            }
#pragma unroll
            for (int c = 0; c < HD / 16; ++c) {
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const Split y = split(*reinterpret_cast<const float*>(stage + G::place(1, half * 8 + t + 4 * (i >> 1), c * 16 + g + 8 * (i & 1))));
                hi[i] = y.hi, lo[i] = y.lo;
              }
#pragma unroll
              for (int n = 0; n < NG; ++n) {
                float y[4] = {};
                mma_tf32(y, lo, p0[n].hi, p1[n].hi);
                mma_tf32(y, hi, p0[n].lo, p1[n].lo);
                mma_tf32(y, hi, p0[n].hi, p1[n].hi);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[n][c][i] += y[i];
              }
            }
          }
        }
      }
      __syncwarp();
      if (i + STAGES < x.count) {
        issue(i + STAGES, slot, st);
        if (i + STAGES + 1 < x.count) slot = look(i + STAGES + 1);
      }
      st = st + 1 == STAGES ? 0 : st + 1;
    }
    // ---- the rows' results
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
    }
    if (!p.joined) {
      // the block's warps have parts of the same item
      __syncthreads();
      float* so = reinterpret_cast<float*>(base);                            // [WARPS][rows][HD], then (maximum, sum)
      float2* sml = reinterpret_cast<float2*>(so + WARPS * rows * HD);
      float* bo = so + WARPS * 8 * NG * (HD + 2);                            // the block's: [rows][HD], then (maximum, sum)
      float2* bml = reinterpret_cast<float2*>(bo + 8 * NG * HD);
      auto write = [&](int r, int ch, float sum, const float (&y)[4]) {
        const int token = r / heads, head = r - token * heads;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;                      // (no key: zeros)
        const float z[4] = {y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv};
        if (ok) Quad<T>::store(static_cast<T*>(a.out) + ((size_t)(x.first + token) * a.nh + h0 + head) * HD + ch, z);
      };
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 8 * n + 2 * t + e;
          if (r >= rows) continue;
          float* to = so + (warp * rows + r) * HD + g;
#pragma unroll
          for (int c = 0; c < HD / 16; ++c) to[c * 16] = o[n][c][e], to[c * 16 + 8] = o[n][c][2 + e];
          if (g == 0) sml[warp * rows + r] = make_float2(m[n][e], l[n][e]);
        }
      __syncthreads();
      for (int i = threadIdx.x; i < rows * (HD / 4); i += THREADS) {
        const int r = i / (HD / 4), ch = (i - r * (HD / 4)) * 4;
        float top = -INFINITY, sum = 0.f, y[4] = {};
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sml[w * rows + r].x);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float2 ml = sml[w * rows + r];
          const float f = fast_exp2(ml.x - ref);
          const float4 v = *reinterpret_cast<const float4*>(so + (w * rows + r) * HD + ch);
          sum += ml.y * f;
          y[0] += v.x * f, y[1] += v.y * f, y[2] += v.z * f, y[3] += v.w * f;
        }
        if (p.cluster > 1) {
          *reinterpret_cast<float4*>(bo + r * HD + ch) = make_float4(y[0], y[1], y[2], y[3]);
          if (ch == 0) bml[r] = make_float2(top, sum);
        } else {
          write(r, ch, sum, y);
        }
      }
      if (p.cluster > 1) {
        // the same over the cluster's blocks, a share of the channels each
        cluster_meet();
        for (int i = (int)blockIdx.x % p.cluster * THREADS + threadIdx.x; i < rows * (HD / 4); i += p.cluster * THREADS) {
          const int r = i / (HD / 4), ch = (i - r * (HD / 4)) * 4;
          const uint32_t at_ml = smem_u32(bml + r), at_o = smem_u32(bo + r * HD + ch);
          float top = -INFINITY, sum = 0.f, y[4] = {};
          float2 ml[8];
          float4 v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            ml[k] = make_float2(-INFINITY, 0.f), v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k >= p.cluster) continue;
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml[k].x), "=f"(ml[k].y) : "r"(in_block(at_ml, k)) : "memory");
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v[k].x), "=f"(v[k].y), "=f"(v[k].z), "=f"(v[k].w) : "r"(in_block(at_o, k)) : "memory");
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k].x);
          const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float f = fast_exp2(ml[k].x - ref);
            sum += ml[k].y * f;
            y[0] += v[k].x * f, y[1] += v[k].y * f, y[2] += v[k].z * f, y[3] += v[k].w * f;
          }
          write(r, ch, sum, y);
        }
        cluster_meet();          // (nobody leaves, or fills its ring again, while another reads it)
      }
      __syncthreads();           // (the ring lies there again)
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      continue;
    }
    if (!ok) continue;
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * n + 2 * t + e;
        if (r >= rows) continue;
        const int token = r / heads;
        const size_t row = (size_t)(x.first + token) * a.nh + h0 + r - token * heads;
        if (x.to == FINAL) {
          const float inv = l[n][e] == 0.f ? 0.f : 1.f / l[n][e];
          T* to = static_cast<T*>(a.out) + row * HD + g;
#pragma unroll
          for (int c = 0; c < HD / 16; ++c)
            to[c * 16] = from_f32<T>(o[n][c][e] * inv), to[c * 16 + 8] = from_f32<T>(o[n][c][2 + e] * inv);
        } else {
          const size_t at = x.to == ROW ? row : x.at * p.rows + r;
          float* to = (x.to == ROW ? p.row_o : x.to == CUT ? p.cut_o : p.far_o) + at * HD + g;
#pragma unroll
          for (int c = 0; c < HD / 16; ++c) to[c * 16] = o[n][c][e], to[c * 16 + 8] = o[n][c][2 + e];
          if (g == 0) (x.to == ROW ? p.row_ml : x.to == CUT ? p.cut_ml : p.far_ml)[at] = make_float2(m[n][e], l[n][e]);
        }
      }
  }
  // (a wait that ran out: nothing may still be on its way into this warp's memory when the block ends)
  if (!ok)
    for (int i = 0; i < STAGES; ++i) wait_bar(&full[i], (phases >> i) & 1u, p.err, 23);
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (!FAR && p.joined) {
    // the joining kernel waits for this launch alone: its first block ends behind the one that ran beside it
    if (p.after && blockIdx.x == 0) pdl_wait();
  }
}

}  // namespace own
}  // namespace
}  // namespace gf
