// One new token's attention over a paged key-value cache of 8 bits (quant_cache.cu: its formulas and
// lay-out), compiled for one head size (-DGF_HEAD_DIM=<multiple of 16, at most 256>).
//
// For a request of `len` tokens the query is the last one, at position p = len - 1; it sees the keys
// first_visible_key(p, span) .. p.  out = sum_c softmax_c(scale <q, K_c>) V_c; a request without a
// token gives zeros.
//
// What bounds it is reading the cache: 2 HD + 8 bytes a key and kv head, used once.  For q, K_c and V_c of one kv head
// that is 2 multiply-adds a byte and query head, far too many for the plain cores and a tenth of what the tensor cores
// do: so both products run there, and a tile of codes becomes operands with as few instructions as possible.
//
//  * S^T = K q^T on mma.sync.m16n8k16 (half precision in, 32-bit sums): 16 keys are the rows, up to 8 query
//    heads of a kv head the columns.  The order of a product's reduction is free as long as both operands
//    share it, so the channels are dealt to the instruction's places such that a thread's places are
//    neighbours in memory: it reads up to 16 bytes of its two keys at a time.
//  * O^T = V^T P^T: the rows are channels, the reduction runs over the 16 keys.  A thread's rows are again
//    chosen to be neighbours in memory; two keys' codes of a channel are put side by side by a byte
//    permutation.  P^T comes from S^T by movmatrix.
//  * Codes become halves exactly: e4m3 by one conversion of two, int8 as 1024 + 128 + code, whose bits are
//    0x64 above the code's, minus 1152; or, for keys, as 2^-24 (code + 128) without any arithmetic, the 128 sum(q)
//    taken off the score.
//  (With 8 query heads a kv head the operands of tcgen05 would be 128 rows of keys that have to be unpacked into
//  shared memory as halves first, four times the bytes that this reads there.)
//
// Half precision holds q and the weights in 11 bits, more than the 8 of a bfloat16 q and result.  A row of q is scaled
// by a power of two so that its largest element is in [2^14, 2^15).  A weight is p times its value row's scale, and these
// are scaled by powers of two, one for all heads that follows the largest value scale and one a head that follows its
// largest weight, such that a head's largest weight so far is above 1 (2^7 as a rule) and all are below 2^15: one that
// is small beside it is off by at most 2^-25 of it.  So neither a large value scale without weight nor a weight without
// value takes bits from the others.  For 32-bit q both are the sum of two halves (22 bits, weights down to 2^-3 after
// scaling; off by 2^-25 below), and tiles' products are added up outside the tensor cores.  Scores, maxima, sums and O
// are 32-bit.
//
// A block is four warps, which take the tiles of its share of the work in turn (how it is shared out: see Cursor),
// each through a ring of two stages of its own: nothing but an item's start and end synchronises the block, and an
// item's first tiles are on their way while the one before is being joined.  Head sizes that are a multiple of 64
// come by TMA, 8 or 16 keys with their values a copy, swizzled so that no read meets another's bank; others, pages
// that are no multiple of 8 and scales that are not aligned come by cp.async.
//
// Measured (bfloat16 q, 4 kv heads of 128 with 7 query heads each, pages of 16, the cache not in L2): 64 requests of
// 4,500 keys on average, 304 MB: 60.1 us, 5.1 TB/s (e4m3; integers 62.4); one request of 131,071 keys, 138 MB: 33.6 us,
// 4.1 TB/s: an SM has blocks for 78 % of the kernel's time (the first tile's chain length -> page -> codes is 4 us, and
// blocks end apart), and the join's launch adds to it.  A ring that only copies reads 6.6 TB/s here, one of cp.async 5.4;
// tiles straight to registers came to 4.0 with the rest of this kernel.
#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "quant.cuh"
#include "tc_common.cuh"

#ifndef GF_HEAD_DIM
#define GF_HEAD_DIM 128
#endif

// (Internal to this library: a static of a template would be shared with the libraries of other head sizes.)
namespace gf {
namespace {

constexpr int HD = GF_HEAD_DIM;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size must be a multiple of 16, <= 256");
constexpr float kLog2E = 1.4426950408889634f;
// Keys of a tile: 32 while their products fit the registers.  What a tile costs beside its bytes (waiting, copies,
// maxima, q from shared memory) is half, and two chains of steps overlap: 304 MB of heads of 128 60 us after 70.
constexpr int TK = HD <= 128 ? 2 : 1, TILE = 16 * TK, TILE_SHIFT = TK == 2 ? 5 : 4;
constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int KW = HD % 64 == 0 ? 16 : HD % 32 == 0 ? 8 : 4;     // bytes of a key a thread reads at once
constexpr int VW = HD % 128 == 0 ? 16 : HD % 64 == 0 ? 8 : HD % 32 == 0 ? 4 : 2;
constexpr int KWORDS = HD / 16;                                  // words of a key a thread holds
constexpr int MT = HD / 16;                                      // row tiles of O^T
constexpr int CH = HD / 16;                                      // 16-byte chunks of a row
// A tile in shared memory.  Head sizes that are a multiple of 64 lie as TMA's swizzle leaves them: rows of SW bytes
// (a wider head is several such tiles), the 16-byte chunks of eight neighbouring rows in turn, so that a quarter
// warp's reads of keys (two rows, four chunks) and of values (four rows, two chunks) hit every bank once (half the
// values of a head of 64: twice).  Others lie in rows 16 bytes apart in banks.
constexpr bool SWIZZLED = HD % 64 == 0;
constexpr int SW = HD % 128 == 0 ? 128 : 64, SUBS = SWIZZLED ? HD / SW : 1, ROW = HD + 16;
constexpr int STAGE = SWIZZLED ? 2 * TILE * HD : 2 * TILE * ROW;
constexpr int SCALES = TILE * 16 + TILE;                         // bytes of a stage's scales
// Keys of a unit (8 or 16 neighbours in a page) are followed by their values: what one TMA copy brings.
struct Layout {
  int eight, values;          // from a row to the one eight behind, from a key to its value
  __device__ __forceinline__ int at(int which, int r, int chunk) const {
    if constexpr (SWIZZLED) {
      const int sub = chunk / (SW / 16), c = chunk % (SW / 16), turn = SW == 128 ? r & 7 : (r >> 1) & 3;
      return sub * (2 * TILE * SW) + (r >> 4) * (32 * SW) + ((r >> 3) & 1) * eight + which * values + (r & 7) * SW +
             ((c ^ turn) << 4);
    } else {
      return (which * TILE + r) * ROW + chunk * 16;
    }
  }
};
constexpr int STAGES = 2;
// Blocks an SM: as many as their registers allow without spilling in a tile's work.  (Two tiles of heads: 52 us with
// two of them, 53 with three, at 16 query heads of 128 a kv head in equal runs; one of heads with 32-bit q: 73 with three,
// 81 with two.)
constexpr int blocks_an_sm(int nt, int type_bytes) {
  return nt == 1 ? (HD <= 64 && type_bytes == 2 ? 4 : 3) : (HD <= 96 ? 3 : 2);
}
// the fewest tiles of a block's run
constexpr int kLeastTiles = 2 * WARPS / TK;
// How the work is shared out (launch_decode).  A cluster of up to kMostOfCluster blocks takes an item where the blocks that
// fit the GPU allow two or more and a request that fills its table keeps them at most as much longer than equal runs would
// as the joining kernel costs, kUnevenKeys keys a block: 8 requests of 576 keys, tables of 4,096, 12 query heads on 2 kv
// heads of 128: 11.1 us after 16.6 with equal runs; one of 8,000 keys, where the rule says equal runs: 16.1 after 19.4.
// kShortKeys keys are one block's work: parts that meet cost more than their keys.  One block / as the rule goes on above it, us,
// full tables of 256 keys: 28 heads on 4 kv heads of 128, one request 7.2 / 8.2, eight 7.4 / 8.3; 14 on 2 of 64, one 6.4 / 6.7,
// 64 6.8 / 8.3; 32 on 2 of 128, eight 9.3 / 10.5; 32-bit q, 28 on 4 of 128, 32 requests 8.2 / 10.8; 8 on 2 of 256, eight
// 10.4 / 9.8; of 384 keys 8.3 / 7.7, 8.6 / 8.2, 7.5 / 6.6, 8.1 / 10.0 (the first four).
// Where there are as many items as SMs, up to kMiddleKeys are one block's, too.  One block / equal runs, us, 28 heads on 4 of 128,
// 128 requests of 102 to 1,024 keys, tables of 1,024 28.0 / 33.1, all full 35.5 / 34.1; to 1,536 36.0 / 38.4, 47.7 / 43.0; to 2,048
// 44.2 / 44.4, 59.3 / 55.1; 14 on 2 of 64, 256 requests, tables of 1,024 19.4 / 25.4, 37.5 / 47.1; 2,048 32.1 / 32.9, 69.5 / 83.7.
constexpr int kShortKeys = 256, kMiddleKeys = 1024, kMostOfCluster = 8, kUnevenKeys = 700;
constexpr int kMostBlocks = 8;          // of the blocks that fit an SM, so many are counted on

struct DecodeArgs {
  const void* q;              // rows of q, or of q | k | v (fused)
  int q_stride;
  uint8_t* codes;
  float* scales;
  const int* block_table;
  int table_stride, limit;    // limit: no request is longer (table width * page)
  int pages;                  // of the cache: an entry of the table beyond it is taken for the nearest
  const int* lengths;
  void* out;
  int out_f32, B, nh, nkv, page, page_shift, span;
  float scale;
  int unit;                   // keys of a TMA copy
  int* err;
  int chunks, rows;           // a kv head's query heads in `chunks` blocks of up to `rows`
  int stream;                 // blocks share the tiles evenly (see Cursor), else `cluster` blocks an item
  int cluster;
  int2* info;                 // [heads * B], stream: the block an item starts in, how many it is spread over
  float* po;                  // [blocks][2][rows][HD]: the parts of the item a block ends in the middle of or starts
  float2* pml;                // [blocks][2][rows]      in the middle of (0: it has begun before this block)
  // the fused step
  const float* table;
  int table_rows, rot, neighbours;
};

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_log2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------------------------------- division of the work
// An item is a (chunk of query heads that share a kv head, request), request by request within a chunk, and its
// tiles are the positions first_visible .. len - 1 cut at multiples of TILE; a request without a token counts as one.
// Where requests are short (DecodeArgs.stream 0) a block takes an item, or a cluster of blocks, which joins its own
// results.  Else the items' tiles are one long sequence, and every block takes an equal run of it: they all end at the same time, whatever the lengths.  A run
// begins and ends inside items; such parts are joined by a second kernel.
__device__ __forceinline__ int request_length(const DecodeArgs& a, int b) {
  return max(min(fresh_index(a.lengths + b), a.limit), 0);
}
__device__ __forceinline__ int first_tile(const DecodeArgs& a, int len) {
  return len > 0 ? first_visible_key(len - 1, a.span) >> TILE_SHIFT : 0;
}
__device__ __forceinline__ int request_tiles(const DecodeArgs& a, int len) {
  return len > 0 ? ((len - 1) >> TILE_SHIFT) - first_tile(a, len) + 1 : 1;
}
struct Cursor {
  int hc, b, len;             // the item
  int off, todo, run;         // tiles of it before this block's, tiles left to this block, tiles a block
};
constexpr int EACH = 4;       // requests a thread keeps in registers
// The run of block `k` of `blocks`, found by the whole block; todo = 0: there is nothing left for it.
__device__ __forceinline__ Cursor find_run(const DecodeArgs& a, int k, int blocks, int heads) {
  __shared__ unsigned counts[WARPS];
  __shared__ Cursor found;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int each = (a.B + THREADS - 1) / THREADS, b0 = threadIdx.x * each, b1 = min(b0 + each, a.B);
  int n[EACH], len[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) len[i] = i < each && b0 + i < b1 ? request_length(a, b0 + i) : -1;
  unsigned mine = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) n[i] = len[i] >= 0 ? request_tiles(a, len[i]) : 0, mine += n[i];
  for (int b = b0 + EACH; b < b1; ++b) mine += request_tiles(a, request_length(a, b));
  unsigned sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  if (lane == 31) counts[warp] = sum;
  if (threadIdx.x == 0) found.todo = 0;
  __syncthreads();
  unsigned start = sum - mine, total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) start += counts[w];
    total += counts[w];
  }
  const unsigned long long all = (unsigned long long)total * heads;
  const bool narrow = all < 0xffff0000ull;         // (64-bit divisions cost more than the rest of this)
  const unsigned long long share = narrow ? ((unsigned)all + blocks - 1) / (unsigned)blocks : (all + blocks - 1) / blocks;
  // (a multiple of the warps, which end together)
  const unsigned long long run = max((share + WARPS - 1) / WARPS * WARPS, (unsigned long long)kLeastTiles), at = run * k;
  if (at < all) {
    const unsigned hc = narrow ? (unsigned)at / total : (unsigned)(at / total);
    const unsigned rest = (unsigned)(at - (unsigned long long)hc * total);
    if (rest >= start && rest < start + mine) {
      int left = (int)(rest - start);
      for (int b = b0; b < b1; ++b) {
        const int i = b - b0, ln = i < EACH ? (i == 0 ? len[0] : i == 1 ? len[1] : i == 2 ? len[2] : len[3])
                                            : request_length(a, b);
        const int tiles = request_tiles(a, ln);
        if (left < tiles) {
          found = {(int)hc, b, ln, left, (int)min(run, all - at), (int)run};
          break;
        }
        left -= tiles;
      }
    }
  }
  __syncthreads();
  return found;
}

// ------------------------------------------------------------------------------------- a tile
template <int BYTES> __device__ __forceinline__ void read_bytes(const uint8_t* p, uint32_t* r);
template <> __device__ __forceinline__ void read_bytes<16>(const uint8_t* p, uint32_t* r) {
  const uint4 x = *reinterpret_cast<const uint4*>(p);
  r[0] = x.x, r[1] = x.y, r[2] = x.z, r[3] = x.w;
}
template <> __device__ __forceinline__ void read_bytes<8>(const uint8_t* p, uint32_t* r) {
  const uint2 x = *reinterpret_cast<const uint2*>(p);
  r[0] = x.x, r[1] = x.y;
}
template <> __device__ __forceinline__ void read_bytes<4>(const uint8_t* p, uint32_t* r) {
  r[0] = *reinterpret_cast<const uint32_t*>(p);
}
template <> __device__ __forceinline__ void read_bytes<2>(const uint8_t* p, uint32_t* r) {
  r[0] = *reinterpret_cast<const uint16_t*>(p);
}
__device__ __forceinline__ void copy16(void* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(dst)), "l"(src),
               "r"(there ? 16 : 0) : "memory");            // (not there: zeros)
}
template <int N> __device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}
// Where a key lies.
struct Place {
  const uint8_t* codes;       // the key's row; its value's lies page * HD behind
  const float2* scales;
};
__device__ __forceinline__ Place place_of(const DecodeArgs& a, int kvh, int page_number, int off) {
  const size_t at = (size_t)page_number * a.nkv + kvh;
  return {a.codes + (at * 2 * a.page + off) * HD, reinterpret_cast<const float2*>(a.scales) + at * a.page + off};
}
__device__ __forceinline__ int page_in(const DecodeArgs& a, int number) {
  return min(max(number, 0), a.pages - 1);
}
__device__ __forceinline__ int logical_page(const DecodeArgs& a, int c) {
  return a.page_shift >= 0 ? c >> a.page_shift : c / a.page;
}
// A warp's view of an item's tiles.
// TMA: pages are a multiple of 8 (unit 8) or 16 (unit 16); a unit comes by one copy of keys and values (for each SW
// bytes of a head) and one of scales, and counts on the stage's barrier.  Lane u knows unit u's page.  Rows that are
// masked come too, and are cleared where they matter (clear_masked).
// Else: lane r knows row r's page, cp.async brings 16 bytes a lane, rows outside [lo, end) are zeros and nothing of
// them is read.
template <bool TMA> struct Tiles {
  const DecodeArgs& a;
  const int* tbl;
  int kvh, lo, end, last, lane;
  Layout lay;
  __device__ __forceinline__ int row_key(int tile, int r) const { return min(max(tile * TILE + r, lo), end - 1); }
  __device__ __forceinline__ int page_of(int tile) const {
    if (tile >= last || lo >= end) return 0;
    return page_in(a, fresh_index(tbl + logical_page(a, row_key(tile, TMA ? (lane * a.unit) & (TILE - 1) : lane & (TILE - 1)))));
  }
  __device__ __forceinline__ void copy(const CUtensorMap* map, uint64_t* bar, uint8_t* stage, uint8_t* scales, int tile,
                                       int page_number) const {
    const int c0 = tile * TILE;
    if constexpr (TMA) {
      const int c = c0 + lane * a.unit;
      const bool mine = lane * a.unit < TILE && c < end && c + a.unit > lo;
      const int units = __popc(__ballot_sync(0xffffffffu, mine));
      if (lane == 0) mbar_expect_tx(bar, units * a.unit * (2 * HD + 8));
      __syncwarp();
      if (mine) {
        const int off = c - logical_page(a, c) * a.page;
#pragma unroll
        for (int sub = 0; sub < SUBS; ++sub)
          asm volatile(
              "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
              "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(stage + sub * (2 * TILE * SW) + lane * a.unit * 2 * SW)),
              "l"(map), "r"(smem_u32(bar)), "r"(sub * SW), "r"(off), "r"(2 * kvh), "r"(page_number)
              : "memory");
        const float2* from = place_of(a, kvh, page_number, off).scales;
        asm volatile(
            "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                smem_u32(scales + lane * a.unit * 8)),
            "l"(from), "r"(a.unit * 8), "r"(smem_u32(bar))
            : "memory");
      }
    } else {
      const size_t values = (size_t)a.page * HD;
      const int c = max(row_key(tile, lane & (TILE - 1)), 0);      // (a row that is masked: one that is there)
      const Place own = place_of(a, kvh, page_number, c - logical_page(a, c) * a.page);
#pragma unroll
      for (int i = 0; i < (TILE * CH + 31) / 32; ++i) {
        const int idx = lane + 32 * i, row = idx / CH, ch = idx - row * CH;
        const bool there = c0 + row >= lo && c0 + row < end;
        const uint8_t* src =
            reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, (unsigned long long)own.codes, row & (TILE - 1))) + ch * 16;
        if (TILE * CH % 32 == 0 || idx < TILE * CH) {
          copy16(stage + lay.at(0, row, ch), src, there);
          copy16(stage + lay.at(1, row, ch), src + values, there);
        }
      }
      // the scales: the 16 bytes that a key's own are in
      if (lane < TILE) {
        const bool there = c0 + lane >= lo && c0 + lane < end;
        const size_t at = (size_t)own.scales;
        const uint32_t odd = (uint32_t)at & 8u;
        if (there && at - odd < (size_t)a.scales)          // (the cache's first ones, where those bytes start before it)
          *reinterpret_cast<float2*>(scales + lane * 16 + 8) = __ldcg(own.scales);
        else
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(scales + lane * 16)),
                       "l"(at - odd), "r"(there ? (odd ? 16 : 8) : 0) : "memory");
        scales[TILE * 16 + lane] = (uint8_t)odd;
      }
    }
  }
  // The (key, value) scales of key r of a tile.
  __device__ __forceinline__ float2 scales(const uint8_t* at, int r) const {
    return *reinterpret_cast<const float2*>(TMA ? at + r * 8 : at + r * 16 + at[TILE * 16 + r]);
  }
  // Masked values count as nothing, whatever lies there (their weight is zero, but zero times no number is none).
  __device__ __forceinline__ void clear_masked(uint8_t* stage, int tile, int len) const {
    if constexpr (TMA) {
      for (int i = lane; i < TILE * CH; i += 32) {
        const int row = i / CH, c = tile * TILE + row;
        if (c < lo || c >= len) *reinterpret_cast<uint4*>(stage + lay.at(1, row, i - row * CH)) = make_uint4(0u, 0u, 0u, 0u);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // (the stage's next copy comes behind this)
      __syncwarp();
    }
  }
};

// The channel that a key's word w of the thread's places t stands for: a quarter of every SW bytes, four a word.
__device__ __forceinline__ constexpr int key_channel(int t, int w) {
  constexpr int SPAN = SWIZZLED ? SW : HD, WORDS = SPAN / 16;
  return w / WORDS * SPAN + t * (SPAN / 4) + w % WORDS * 4;
}
// Where channel c of head r stands in a block's q (see quant_decode_kernel).
__device__ __forceinline__ int q_place(int r, int c) {
  constexpr int SPAN = SWIZZLED ? SW : HD, WORDS = SPAN / 16;
  const int in = c % SPAN, t = in / (SPAN / 4), w = c / SPAN * WORDS + in % (SPAN / 4) / 4;
  return (((r >> 3) * KWORDS + w) * 32 + (r & 7) * 4 + t) * 4 + (c & 3);
}
// Two codes plus 128 (the bytes 2i, 2i + 1 of a word) as the halves 2^-24 (code + 128), below the smallest normal one:
// a byte permutation, no arithmetic.
__device__ __forceinline__ uint32_t raised_halves(uint32_t w, int i) {
  return __byte_perm(w, 0u, i ? 0x4342 : 0x4140);
}
// Two codes in the bytes 2i, 2i + 1 of a word, as two halves.
template <bool FP8> __device__ __forceinline__ uint32_t halves(uint32_t w, int i) {
  if constexpr (FP8) {
    return e4m3x2_to_half2(i ? w >> 16 : w);
  } else {                                         // (w: the codes plus 128)
    const uint32_t r = __byte_perm(w, 0x64646464u, i ? 0x4342 : 0x4140);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&r), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// what a float loses when it is rounded to a half
__device__ __forceinline__ float half_rest(float x) { return x - __half2float(__float2half_rn(x)); }
// p is 2^(score - m).  m + h, h of a head as a rule 0, is the whole number kSlack above the largest score that there was when
// it was raised last.  Weights are p times a value's scale times 2^(f - 127), where f = kSafe - e with the largest
// (biased) exponent e of the scales: below 2^15 for every p up to 1, and the largest at 2^7 or 2^6 when m is raised, if its
// scale is the largest too.  Where the largest weight of a head would be below 1, its h takes it to [1, 2).
constexpr float kSlack = 7.f;
constexpr int kSafe = 127 + 127 + 14, kMostExtra = 100;
// 2^(127 - f) for 7 <= f <= 254
__device__ __forceinline__ float power_back(int f) {
  return __uint_as_float(f == 254 ? 0x00400000u : (uint32_t)(254 - f) << 23);
}
// The bits of the first power of two that is too large a scale for a weight of p = 1 and f (with its head's h).
__device__ __forceinline__ uint32_t scale_limit(int f) { return (uint32_t)min(kSafe + 1 - f, 255) << 23; }

// ------------------------------------------------------------------------------------- q, and the new token
// A lane's channels of head rows: lane, lane + 32, ...  Everything is asked for before anything is used.
constexpr int N = (HD + 31) / 32;
template <typename T> __device__ __forceinline__ float row_value(const DecodeArgs& a, size_t at) {
  return fresh(reinterpret_cast<const T*>(a.q) + at);
}
template <typename T>
__device__ __forceinline__ void load_row(const DecodeArgs& a, size_t at, bool there, int lane, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = there && i * 32 + lane < HD ? row_value<T>(a, at + i * 32 + lane) : 0.f;
}
// The channel that channel c turns with, and which of the pair c is.
__device__ __forceinline__ int partner(const DecodeArgs& a, int c, bool& second) {
  const int half = a.rot >> 1;
  second = a.neighbours ? (c & 1) : c >= half;
  return a.neighbours ? c ^ 1 : second ? c - half : c + half;
}
struct Angles {
  float c[N], s[N];                        // a first of a pair takes off what a second adds: -s
  __device__ __forceinline__ void load(const DecodeArgs& a, int p, int lane) {
    const float* cs = a.table + (size_t)min(p, a.table_rows - 1) * a.rot;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int ch = i * 32 + lane, half = a.rot >> 1;
      const int j = a.neighbours ? ch >> 1 : ch >= half ? ch - half : ch;
      c[i] = ch < a.rot ? __ldg(cs + j) : 1.f;
      const float sine = ch < a.rot ? __ldg(cs + half + j) : 0.f;
      s[i] = (a.neighbours ? ch & 1 : ch >= half) ? sine : -sine;
    }
  }
};
// Where they turn in halves of a whole head or with neighbours, a channel's partner is in the warp's registers.
__device__ __forceinline__ bool partners_here(const DecodeArgs& a) {
  return a.rot == 0 || (HD % 64 == 0 && a.rot == HD && !a.neighbours) || a.neighbours;
}
__device__ __forceinline__ void take_partners(const DecodeArgs& a, const float (&x)[N], float (&y)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float n = __shfl_xor_sync(0xffffffffu, x[i], 1);
    y[i] = a.neighbours ? n : x[N % 2 ? i : i < N / 2 ? i + N / 2 : i - N / 2];
  }
}
template <typename T>
__device__ __forceinline__ void load_partners(const DecodeArgs& a, size_t at, bool there, int lane, float (&y)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    bool second;
    const int c = i * 32 + lane;
    y[i] = there && c < a.rot ? row_value<T>(a, at + partner(a, c, second)) : 0.f;
  }
}
__device__ __forceinline__ void turn_row(const DecodeArgs& a, const Angles& an, int lane, float (&x)[N], const float (&y)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i * 32 + lane < a.rot) x[i] = __fadd_rn(__fmul_rn(x[i], an.c[i]), __fmul_rn(y[i], an.s[i]));
}
__device__ __forceinline__ uint32_t row_top(const float (&x)[N]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  return group_max_bits<32>(top);
}

// ------------------------------------------------------------------------------------- a block's run
// Floats from a head's result to the next one's in shared memory: two rows in other banks, unless a warp's results then no
// longer fit a stage.
__host__ __device__ constexpr int result_row(int nt) {
  return 8 * nt * (HD + 2) * 4 > STAGE && 8 * nt * HD * 4 <= STAGE ? HD : HD + 2;
}
struct Item {
  int b, hc, len, lo, first, last;         // its tiles here
  bool starts, ends;                       // whether they are its first, its last
};
// What a block goes on with behind an item's tiles.
struct Kept {
  Item next, done;
  Cursor cur;
  int soon_b, soon_len;
};
// NT: tiles of 8 query heads.  T: the type of q and the result (32-bit ones take two halves each).  STEP: q | k | v
// rows, unrotated.
template <int NT, bool FP8, typename T, bool TMA, bool STEP>
__global__ void __launch_bounds__(THREADS, blocks_an_sm(NT, sizeof(T)))
quant_decode_kernel(const DecodeArgs a, const __grid_constant__ CUtensorMap map) {
  constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
  constexpr int R = 8 * NT, RW = R / WARPS;                      // rows of q in all, and a warp
  constexpr bool RAISED = !FP8 && PARTS == 1;                    // K's codes as halves of code + 128
  constexpr int OROW = result_row(NT);
  // [WARPS][STAGES][STAGE], [WARPS][STAGES][SCALES]; a warp's results at an item's end go into its stage that is not under
  // way, or where that is too small behind the ring
  extern __shared__ uint8_t raw[];
  uint8_t* ring = raw + ((0u - smem_u32(raw)) & 1023u);          // (a swizzle counts from 1 KB)
  constexpr bool IN_STAGE = R * OROW * 4 <= STAGE;
  // q as the products want it: [half][tile of heads][word of a key][lane][four channels]; read again for every tile,
  // so that four blocks' registers fit an SM
  __shared__ __align__(16) __half qh[PARTS][NT][KWORDS][32][4];
  // a score is (product * x + y) * the key's scale
  __shared__ __align__(16) float2 q_back[R];
  __shared__ float sm[WARPS][R], sl[WARPS][R], back[WARPS];
  __shared__ int so_at[WARPS];
  __shared__ __align__(16) uint8_t fresh_row[2][HD];             // STEP: the new token's codes and scales
  __shared__ float fresh_scale[2];
  __shared__ uint64_t bars[WARPS][STAGES];
  __shared__ Kept kept[WARPS];
  __shared__ int parts_of_item;                                  // a cluster's
  if (TMA && threadIdx.x == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(&map) : "memory");
  if (TMA && (threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < STAGES; ++i) mbar_init(&bars[threadIdx.x >> 5][i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncwarp();
  if (a.stream) {
    // what an item's start waits for comes from far off (the cache has swept it out of L2): asked for early
    const auto ask = [](const void* at) { asm volatile("prefetch.global.L2 [%0];" ::"l"(at)); };
    const long long i = (long long)blockIdx.x * THREADS + threadIdx.x;
    if (i * 32 < a.B) ask(a.lengths + i * 32);
    if (i * 32 < (long long)a.B * a.table_stride) ask(a.block_table + i * 32);
    constexpr int LINE = 128 / sizeof(T);
    const long long lines = a.nh * HD / LINE;
    if (i < a.B * lines) ask(reinterpret_cast<const T*>(a.q) + (size_t)(i / lines) * a.q_stride + (i % lines) * LINE);
  }
  pdl_wait();
  const int heads = a.nkv * a.chunks, G = a.nh / a.nkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* mine = ring + warp * STAGES * STAGE;
  uint8_t* my_scales = ring + WARPS * STAGES * STAGE + warp * STAGES * SCALES;
  const Layout lay = {TMA && a.unit == 8 ? 16 * SW : 8 * SW, TMA && a.unit == 8 ? 8 * SW : 16 * SW};
  uint32_t phases = 0;                     // of the stages' barriers, a bit each
  bool lost = false;                       // a copy has not come within the limit: nothing more is waited for
  Cursor cur;
  // The joining kernel is let in early only where this one leaves SMs idle: else its waiting blocks take the places of
  // the next call's, which then start late (12 us of 76 with 592 blocks).
  if (!a.stream) pdl_trigger();
  if (a.stream) {
    cur = find_run(a, blockIdx.x, gridDim.x, heads);
    if (cur.todo == 0 || cur.run == kLeastTiles) pdl_trigger();
  } else {
    const int item = blockIdx.x / a.cluster, rank = blockIdx.x - item * a.cluster;
    cur.b = item / heads, cur.hc = item - cur.b * heads, cur.len = request_length(a, cur.b);
    const int n = request_tiles(a, cur.len);
    cur.run = ((n + a.cluster - 1) / a.cluster + WARPS - 1) / WARPS * WARPS;
    cur.off = rank * cur.run, cur.todo = max(min(n - cur.off, cur.run), 0);
    if (threadIdx.x == 0) parts_of_item = (n + cur.run - 1) / cur.run;
  }
  const auto head_of = [&](int hc) { return (hc / a.chunks) * G + (hc % a.chunks) * a.rows; };
  const auto rows_of = [&](int hc) { return min(a.rows, G - (hc % a.chunks) * a.rows); };
  // The block's next item that has tokens; the others get their zeros.
  // lengths on their way: of the request that the cursor will be on after this item, and of the one behind that
  int soon_b = -1, soon_len = 0, later_b = -1, later_len = 0;
  const auto next_item = [&](Item& it) {
    while (cur.todo > 0) {
      const int len = cur.len, t0 = first_tile(a, len), n = request_tiles(a, len);
      it.b = cur.b, it.hc = cur.hc, it.len = len, it.lo = len > 0 ? first_visible_key(len - 1, a.span) : 0;
      it.first = t0 + cur.off, it.last = it.first + min(n - cur.off, cur.todo);
      it.starts = cur.off == 0, it.ends = it.last == t0 + n;
      if (a.stream && it.starts && threadIdx.x == 0)
        a.info[it.hc * a.B + it.b] = make_int2(blockIdx.x, 1 + (t0 + n - it.last + cur.run - 1) / cur.run);
      cur.todo -= it.last - it.first, cur.off = 0;
      if (++cur.b == a.B) cur.b = 0, ++cur.hc;
      if (len > 0) return true;
      for (int i = threadIdx.x; i < rows_of(it.hc) * HD; i += THREADS)
        reinterpret_cast<T*>(a.out)[((size_t)it.b * a.nh + head_of(it.hc)) * HD + i] = from_f32<T>(0.f);
      if (cur.todo > 0) cur.len = request_length(a, cur.b);
    }
    return false;
  };

  int pages[STAGES];
  const auto tiles_of = [&](const Item& it) {
    return Tiles<TMA>{a, a.block_table + (size_t)it.b * a.table_stride, it.hc / a.chunks, it.lo,
                      STEP && !TMA ? it.len - 1 : it.len, it.last, lane, lay};
  };
  const auto ask_pages = [&](const Item& it) {
#pragma unroll
    for (int i = 0; i < STAGES; ++i) pages[i] = tiles_of(it).page_of(it.first + warp + i * WARPS);
  };

  float o[NT][MT][4], m[NT][2], l[NT][2];
  int f = 254;                             // weights are multiplied by 2^(f - 127)
  uint32_t extra = 0, too_large = 0;       // the heads' h, 8 bits each; scale_limit of f and the largest of them
  int at_stage = 0, to_stage = STAGES - 1;
  Item it;
  bool have = next_item(it), had = false;
  if (have) ask_pages(it);
  if (cur.todo > 0) soon_b = cur.b, soon_len = request_length(a, cur.b);
  while (true) {
    // ---- an item's start: all that it waits for is asked for before anything is used
    const int kvh = it.hc / a.chunks, h0 = head_of(it.hc), nrows = rows_of(it.hc), p = it.len - 1;
    const size_t row = (size_t)it.b * a.q_stride;
    const Tiles<TMA> tiles = tiles_of(it);
    float x[RW][N], y[RW][N], nx[N], ny[N];
    Angles an;
    // the new token's row of keys (the last warp's, whose rows of q may not exist) and of values (the one before)
    const bool news = STEP && it.ends && warp >= WARPS - 2, keys = warp == WARPS - 1;
    int new_page = 0, page_number = 0;
    if (have) {
#pragma unroll
      for (int i = 0; i < RW; ++i)
        load_row<T>(a, row + (size_t)(h0 + warp + i * WARPS) * HD, warp + i * WARPS < nrows, lane, x[i]);
      if constexpr (STEP) {
        an.load(a, p, lane);
        const size_t new_at = row + (size_t)(a.nh + (keys ? 0 : a.nkv) + kvh) * HD;
        if (news) load_row<T>(a, new_at, true, lane, nx);
        if (!partners_here(a)) {
#pragma unroll
          for (int i = 0; i < RW; ++i)
            load_partners<T>(a, row + (size_t)(h0 + warp + i * WARPS) * HD, warp + i * WARPS < nrows, lane, y[i]);
          if (news && keys) load_partners<T>(a, new_at, true, lane, ny);
        }
        // (an entry that is no page, or a token behind the table's end: nowhere to write it to)
        if (news) new_page = fresh_index(tiles.tbl + logical_page(a, p));
        if (news && it.len == a.limit && fresh_index(a.lengths + it.b) > a.limit) new_page = -1;
      }
      if (cur.todo > 0) later_b = cur.b + 1 == a.B ? 0 : cur.b + 1, later_len = request_length(a, later_b);
      // (of the new token nothing is read)
      int stage = at_stage;
#pragma unroll
      for (int i = 0; i < STAGES - 1; ++i) {
        const int tile = it.first + warp + i * WARPS;
        if (tile < it.last && !lost) tiles.copy(&map, &bars[warp][stage], mine + stage * STAGE, my_scales + stage * SCALES, tile, pages[i]);
        if constexpr (!TMA) asm volatile("cp.async.commit_group;\n");
        stage = stage + 1 == STAGES ? 0 : stage + 1;
      }
      page_number = pages[STAGES - 1];
    }

    if (!have) pdl_trigger();
    // ---- the end of the item before: the four warps' results
    if (had) {
      const Item done = kept[warp].done;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 4);
          l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 8);
          l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 16);
          if (g == 0) sm[warp][n * 8 + 2 * t + j] = m[n][j], sl[warp][n * 8 + 2 * t + j] = l[n][j];
        }
      const int place = IN_STAGE ? (warp * STAGES + to_stage) * STAGE : WARPS * STAGES * (STAGE + SCALES) + warp * R * OROW * 4;
      if (lane == 0) back[warp] = power_back(f), so_at[warp] = place;
      __syncwarp();                        // (the stage's tile has been read)
      float* so = reinterpret_cast<float*>(ring + place);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        constexpr int STEP_W = VW >= 4 ? VW / 4 : 1, PER = VW >= 4 ? 2 : 1;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int w = i / PER;
          const int c = ((w / STEP_W) * 8 + g) * VW + (w % STEP_W) * 4 + (i % PER) * 2;
          float* at = so + (n * 8 + 2 * t) * OROW + c;
          *reinterpret_cast<float2*>(at) = make_float2(o[n][i][0], o[n][i][2]);
          *reinterpret_cast<float2*>(at + OROW) = make_float2(o[n][i][1], o[n][i][3]);
        }
      }
      if constexpr (TMA && IN_STAGE) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncthreads();
      const bool whole = done.starts && done.ends;
      const size_t part = ((size_t)blockIdx.x * 2 + (done.starts ? 1 : 0)) * a.rows;
      const size_t out_at = ((size_t)done.b * a.nh + head_of(done.hc)) * HD;
      const int n_out = rows_of(done.hc) * (HD / 2);
#pragma unroll 1
      for (int i = threadIdx.x; i < n_out; i += THREADS) {
        const int r = i / (HD / 2), c = 2 * (i - r * (HD / 2));
        float top = sm[0][r];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) top = fmaxf(top, sm[w][r]);
        float sum = 0.f, v0 = 0.f, v1 = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          // (a warp without tiles has sums of zero; one whose scores are no numbers passes that on)
          const float e = sm[w][r] == -INFINITY ? 0.f : fast_exp2(sm[w][r] - top), b = back[w];
          const float2 v = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(ring + so_at[w]) + r * OROW + c);
          sum += e * sl[w][r], v0 += e * v.x * b, v1 += e * v.y * b;
        }
        const float inv = __fdividef(1.f, sum);
        v0 *= inv, v1 *= inv;
        if (!whole) {
          *reinterpret_cast<float2*>(a.po + (part + r) * HD + c) = make_float2(v0, v1);
          if (c == 0) a.pml[part + r] = make_float2(top, sum);
        } else if constexpr (sizeof(T) == 4) {
          *reinterpret_cast<float2*>(reinterpret_cast<float*>(a.out) + out_at + 2 * i) = make_float2(v0, v1);
        } else {
          *reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<bf16*>(a.out) + out_at + 2 * i) = __floats2bfloat162_rn(v0, v1);
        }
      }
    }
    if (!have) break;

    // ---- q, and the new token
    if constexpr (STEP) {
      // The block that has the item's last tile writes the new token (every chunk of heads the same bytes) and
      // keeps it for its own tile.
      if (news) {
        if (keys) {
          if (partners_here(a)) take_partners(a, nx, ny);
          turn_row(a, an, lane, nx, ny);
        }
        const RowScale rs = row_scale(row_top(nx), FP8);
        const Place pl = place_of(a, kvh, page_in(a, new_page), p - logical_page(a, p) * a.page);
        const int which = keys ? 0 : 1;
        uint8_t* dst = const_cast<uint8_t*>(pl.codes) + (size_t)which * a.page * HD;
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (i * 32 + lane < HD) fresh_row[which][i * 32 + lane] = (uint8_t)code_of(nx[i], rs, FP8);
        if (lane == 0) fresh_scale[which] = rs.scale;
        if (new_page == page_in(a, new_page)) {
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (i * 32 + lane < HD) dst[i * 32 + lane] = fresh_row[which][i * 32 + lane];
          if (lane == 0) reinterpret_cast<float*>(const_cast<float2*>(pl.scales))[which] = rs.scale;
        }
      }
#pragma unroll
      for (int i = 0; i < RW; ++i) {
        if (partners_here(a)) take_partners(a, x[i], y[i]);
        turn_row(a, an, lane, x[i], y[i]);
      }
    }
    // q in halves, a row's largest element in [2^14, 2^15)
#pragma unroll
    for (int j = 0; j < RW; ++j) {
      const int r = warp + j * WARPS;
      const uint32_t top = row_top(x[j]);
      // 2^up takes the largest element to [2^14, 2^15); what is no number stays none
      const int e = top >= 0x7f800000u ? 127 : max((int)(top >> 23), 1), up = min(127 + 14 - e, 126);
      const float scale_up = __uint_as_float((uint32_t)(127 + up) << 23);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = i * 32 + lane;
        if (c < HD) {
          const int at = q_place(r, c);
          (&qh[0][0][0][0][0])[at] = __float2half_rn(x[j][i] * scale_up);
          if constexpr (RAISED) sum += __half2float(__float2half_rn(x[j][i] * scale_up));
          if constexpr (PARTS == 2) (&qh[PARTS - 1][0][0][0][0])[at] = __float2half_rn(half_rest(x[j][i] * scale_up));
        }
      }
      if constexpr (RAISED) sum = warp_sum(sum);
      if (lane == 0) {
        const float qs = a.scale * kLog2E * __uint_as_float((uint32_t)(127 - up) << 23);
        q_back[r] = make_float2(RAISED ? qs * 16777216.f : qs, -128.f * sum * qs);
      }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        m[n][j] = -INFINITY, l[n][j] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }
    f = 254, extra = 0, too_large = scale_limit(254);

    // ---- where the block goes next (its pages are there when this item's tiles are done)
    const Item done = it;
    had = true;
    const int lo = it.lo, len = it.len, last = it.last, first = it.first;
    if (cur.todo > 0) cur.len = soon_b == cur.b ? soon_len : request_length(a, cur.b);
    have = next_item(it);
    soon_b = later_b, soon_len = later_len;
    if (lane == 0) kept[warp] = {it, done, cur, soon_b, soon_len};       // (no use of registers for it meanwhile)
    __syncwarp();
    if (have) ask_pages(it);
    if constexpr (STEP) {      // (the angles of that item's position)
      const float* cs = a.table + (size_t)min(max(it.len - 1, 0), a.table_rows - 1) * a.rot;
      if (have && threadIdx.x * 32 < a.rot) asm volatile("prefetch.global.L2 [%0];" ::"l"(cs + threadIdx.x * 32));
    }

    // ---- the tiles
#pragma unroll 1
    for (int tile = first + warp; tile < last && !lost; tile += WARPS) {
      if constexpr (TMA) {
        lost = !mbar_wait(&bars[warp][at_stage], phases >> at_stage & 1u, a.err, 1);
        lost = __any_sync(0xffffffffu, lost);
        if (lost) {            // (what is under way must not find another block's shared memory)
#pragma unroll 1
          for (int i = 0; i < STAGES - 1; ++i) {
            const int st = (at_stage + i) % STAGES;
            if (tile + i * WARPS < last) mbar_wait(&bars[warp][st], phases >> st & 1u, nullptr, 0);
          }
          break;
        }
        phases ^= 1u << at_stage;
      } else {
        wait_copies<STAGES - 2>();
      }
      __syncwarp();            // every lane's copies have landed, and the stage before has been read
      uint8_t* stage = mine + at_stage * STAGE;
      const uint8_t* stage_scales = my_scales + at_stage * SCALES;
      const int c0 = tile * TILE;
      {
        const int far = tile + (STAGES - 1) * WARPS;
        const int next_page = tiles.page_of(far + WARPS);
        if (far < last)
          tiles.copy(&map, &bars[warp][to_stage], mine + to_stage * STAGE, my_scales + to_stage * SCALES, far, page_number);
        if constexpr (!TMA) asm volatile("cp.async.commit_group;\n");
        page_number = next_page;
      }
      at_stage = at_stage + 1 == STAGES ? 0 : at_stage + 1;
      to_stage = to_stage + 1 == STAGES ? 0 : to_stage + 1;
      float2 sc[2 * TK];           // of keys g, g + 8, ...
#pragma unroll
      for (int i = 0; i < 2 * TK; ++i) sc[i] = tiles.scales(stage_scales, g + 8 * i);
      const bool edge = c0 < lo || c0 + TILE > len;
      if (edge) tiles.clear_masked(stage, tile, len);
      if constexpr (STEP) {
        if (c0 + TILE >= len) {     // the tile of the new token
          const int r = len - 1 - c0;
          for (int i = lane; i < 2 * CH; i += 32) {
            const int which = i / CH, ch = i - which * CH;
            *reinterpret_cast<uint4*>(stage + lay.at(which, r, ch)) =
                *reinterpret_cast<const uint4*>(&fresh_row[which][ch * 16]);
          }
          if constexpr (TMA) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          const float2 mine_sc = make_float2(fresh_scale[0], fresh_scale[1]);
#pragma unroll
          for (int i = 0; i < 2 * TK; ++i)
            if (g + 8 * i == r) sc[i] = mine_sc;
        }
      }
      // S^T, in two chains of products for each 16 keys
      constexpr int CHAINS = KWORDS > 1 ? 2 : 1;
      float s[TK][NT][4];
#pragma unroll
      for (int q = 0; q < TK; ++q) {
        float s2[CHAINS][NT][4];
#pragma unroll
        for (int c = 0; c < CHAINS; ++c)
#pragma unroll
          for (int n = 0; n < NT; ++n) s2[c][n][0] = s2[c][n][1] = s2[c][n][2] = s2[c][n][3] = 0.f;
        uint32_t k[2][KWORDS];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < KWORDS / (KW / 4); ++j)
            read_bytes<KW>(stage + lay.at(0, 16 * q + 8 * i + g, key_channel(t, j * (KW / 4)) / 16) +
                               key_channel(t, j * (KW / 4)) % 16, &k[i][j * (KW / 4)]);
#pragma unroll
        for (int w = 0; w < KWORDS; ++w) {
          const uint32_t k0 = FP8 ? k[0][w] : k[0][w] ^ 0x80808080u, k1 = FP8 ? k[1][w] : k[1][w] ^ 0x80808080u;
          uint32_t A[4];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            A[2 * i] = RAISED ? raised_halves(k0, i) : halves<FP8>(k0, i);
            A[2 * i + 1] = RAISED ? raised_halves(k1, i) : halves<FP8>(k1, i);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = PARTS - 1; i >= 0; --i) {
              const uint2 two = *reinterpret_cast<const uint2*>(&qh[i][n][w][lane][0]);
              mma_f16(s2[w % CHAINS][n], A, two.x, two.y);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[q][n][e] = CHAINS == 2 ? s2[0][n][e] + s2[CHAINS - 1][n][e] : s2[0][n][e];
      }
      bool seen[2 * TK];
#pragma unroll
      for (int i = 0; i < 2 * TK; ++i) seen[i] = true;
      if (edge) {
        // masked keys: whatever lies there counts as nothing (their codes are zeros already)
#pragma unroll
        for (int i = 0; i < 2 * TK; ++i) {
          const int c = c0 + g + 8 * i;
          seen[i] = c >= lo && c < len;
          if (!seen[i]) sc[i] = make_float2(0.f, 0.f);
        }
      }
      // Scores in units of log2.  m, f and h are looked at again only when a score is above m, or a value's scale too
      // large for a p of 1.
      bool above = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float4 qb = *reinterpret_cast<const float4*>(&q_back[n * 8 + 2 * t]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < 2 * TK; ++i) {
            float& r = s[i >> 1][n][2 * (i & 1) + j];
            r = RAISED ? fmaf(r, j ? qb.z : qb.x, j ? qb.w : qb.y) : r * (j ? qb.z : qb.x);
            r = seen[i] ? r * sc[i].x : -INFINITY;
            top = fmaxf(top, r);
          }
          above |= top > m[n][j];
        }
      }
      uint32_t vtop = 0;
#pragma unroll
      for (int i = 0; i < 2 * TK; ++i) {
        const uint32_t bits = __float_as_uint(sc[i].y);
        vtop = max(vtop, bits < 0x7f800000u ? bits : 0u);
      }
      above |= vtop >= too_large;
      if (__any_sync(0xffffffffu, above)) {
        const int f_new = min(f, kSafe - (int)(__reduce_max_sync(0xffffffffu, vtop) >> 23));
        float size[2 * TK];
#pragma unroll
        for (int i = 0; i < 2 * TK; ++i) size[i] = fast_log2(sc[i].y);
        uint32_t h_new = 0, h_most = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float corr[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float top = -INFINITY, weight = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2 * TK; ++i) {
              const float r = s[i >> 1][n][2 * (i & 1) + j];
              top = fmaxf(top, r), weight = fmaxf(weight, r + size[i]);
            }
#pragma unroll
            for (int lanes = 4; lanes <= 16; lanes *= 2) {
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, lanes));
              weight = fmaxf(weight, __shfl_xor_sync(0xffffffffu, weight, lanes));
            }
            const int h = extra >> (8 * (2 * n + j)) & 255u;
            const float highest = m[n][j] + (float)h, mn = top > highest ? ceilf(top + kSlack) : highest;
            const float rise = mn == highest ? 0.f : mn - highest;
            // what the weights so far lose, in whole powers of two, h may give them; need is what takes this tile's
            // largest to [1, 2)
            const int need = 127 - (int)floorf(fminf(fmaxf(weight - mn, -127.f), 120.f));
            const int both = min((int)fminf((float)(f + h) + rise, (float)(f_new + kMostExtra)), max(f_new, need));
            const uint32_t now = (uint32_t)(both - f_new);
            const float to = mn - (float)now, less = to == m[n][j] ? 0.f : m[n][j] - to;
            l[n][j] *= fast_exp2(less);
            corr[j] = fast_exp2(less + (float)(f_new - f));
            m[n][j] = to;
            h_new |= now << (8 * (2 * n + j)), h_most = max(h_most, now);
          }
#pragma unroll
          for (int i = 0; i < MT; ++i)
            o[n][i][0] *= corr[0], o[n][i][1] *= corr[1], o[n][i][2] *= corr[0], o[n][i][3] *= corr[1];
        }
        f = f_new, extra = h_new, too_large = scale_limit(f + (int)h_most);
      }
      const float up = __uint_as_float((uint32_t)f << 23);
      uint32_t P[TK][PARTS][NT][2];
#pragma unroll
      for (int q = 0; q < TK; ++q) {
        const float vs0 = sc[2 * q].y * up, vs1 = sc[2 * q + 1].y * up;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float w[4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float p0 = fast_exp2(s[q][n][j] - m[n][j]), p1 = fast_exp2(s[q][n][2 + j] - m[n][j]);
            l[n][j] += p0 + p1;
            w[j] = p0 * vs0, w[2 + j] = p1 * vs1;
          }
          P[q][0][n][0] = transposed(pack_half(w[0], w[1]));
          P[q][0][n][1] = transposed(pack_half(w[2], w[3]));
          if constexpr (PARTS == 2) {
            P[q][PARTS - 1][n][0] = transposed(pack_half(half_rest(w[0]), half_rest(w[1])));
            P[q][PARTS - 1][n][1] = transposed(pack_half(half_rest(w[2]), half_rest(w[3])));
          }
        }
      }
#pragma unroll
      for (int j = 0; j < HD / (8 * VW); ++j) {
        constexpr int WORDS = VW >= 4 ? VW / 4 : 1, PER = VW >= 4 ? 2 : 1;
        float d[WORDS * PER][NT][4];       // 32-bit results: a tile's products are added up outside the tensor cores
        if constexpr (PARTS == 2)
#pragma unroll
          for (int i = 0; i < WORDS * PER; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) d[i][n][0] = d[i][n][1] = d[i][n][2] = d[i][n][3] = 0.f;
#pragma unroll
        for (int q = 0; q < TK; ++q) {
          uint32_t v[4][WORDS];            // keys 2t, 2t + 1, 2t + 8, 2t + 9 of the 16
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            read_bytes<VW>(stage + lay.at(1, 16 * q + 8 * (i >> 1) + 2 * t + (i & 1), (j * 8 + g) * VW / 16) +
                               (j * 8 + g) * VW % 16, v[i]);
            if constexpr (!FP8) {
#pragma unroll
              for (int w = 0; w < WORDS; ++w) v[i][w] ^= 0x80808080u;
            }
          }
#pragma unroll
          for (int w = 0; w < WORDS; ++w)
#pragma unroll
            for (int y = 0; y < PER; ++y) {
              const uint32_t u0 = __byte_perm(v[0][w], v[1][w], y ? 0x7362 : 0x5140);
              const uint32_t u1 = __byte_perm(v[2][w], v[3][w], y ? 0x7362 : 0x5140);
              const uint32_t A[4] = {halves<FP8>(u0, 0), halves<FP8>(u0, 1), halves<FP8>(u1, 0), halves<FP8>(u1, 1)};
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                if constexpr (PARTS == 2) {
                  mma_f16(d[w * PER + y][n], A, P[q][1][n][0], P[q][1][n][1]);
                  mma_f16(d[w * PER + y][n], A, P[q][0][n][0], P[q][0][n][1]);
                } else {
                  mma_f16(o[n][(j * WORDS + w) * PER + y], A, P[q][0][n][0], P[q][0][n][1]);
                }
              }
            }
        }
        if constexpr (PARTS == 2)
#pragma unroll
          for (int i = 0; i < WORDS * PER; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[n][j * WORDS * PER + i][e] += d[i][n][e];
      }
    }
    it = kept[warp].next, cur = kept[warp].cur;
    soon_b = kept[warp].soon_b, soon_len = kept[warp].soon_len;
    __syncwarp();
  }
  // ---- a cluster's parts, every block a share of the channels
  if (!a.stream && a.cluster > 1) {
    __syncwarp();
    cluster_sync();
    const int parts = parts_of_item, item = blockIdx.x / a.cluster, rank = blockIdx.x - item * a.cluster;
    if (parts == 1) return;
    const int b = item / heads, hc = item - b * heads, n_out = rows_of(hc) * (HD / 2);
    const size_t out_at = ((size_t)b * a.nh + head_of(hc)) * HD, part0 = (size_t)item * a.cluster * 2;
    for (int i = rank * THREADS + threadIdx.x; i < n_out; i += a.cluster * THREADS) {
      const int r = i / (HD / 2), c = 2 * (i - r * (HD / 2));
      float2 ml[kMostOfCluster], v[kMostOfCluster];
#pragma unroll
      for (int k = 0; k < kMostOfCluster; ++k) {
        ml[k] = make_float2(-INFINITY, 0.f), v[k] = make_float2(0.f, 0.f);
        if (k < parts) {
          const size_t part = (part0 + (k ? 2 * k : 1)) * a.rows + r;
          ml[k] = __ldcg(a.pml + part), v[k] = __ldcg(reinterpret_cast<const float2*>(a.po + part * HD + c));
        }
      }
      float top = ml[0].x, sum = 0.f, v0 = 0.f, v1 = 0.f;
#pragma unroll
      for (int k = 1; k < kMostOfCluster; ++k) top = fmaxf(top, ml[k].x);
#pragma unroll
      for (int k = 0; k < kMostOfCluster; ++k) {
        // (a part whose scores are no numbers has a maximum of -inf and passes its sum on)
        const float w = (ml[k].x == -INFINITY ? 0.f : fast_exp2(ml[k].x - top)) * ml[k].y;
        sum += w, v0 = fmaf(w, v[k].x, v0), v1 = fmaf(w, v[k].y, v1);
      }
      const float inv = 1.f / sum;
      if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float2*>(reinterpret_cast<float*>(a.out) + out_at + 2 * i) = make_float2(v0 * inv, v1 * inv);
      else
        *reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<bf16*>(a.out) + out_at + 2 * i) =
            __floats2bfloat162_rn(v0 * inv, v1 * inv);
    }
  }
}

// A block an item and `gridDim.y`-th of its heads: the pieces' results, weighted by their shares of the sum.
// A team of HD / 4 threads takes a head where there are few pieces, else every TEAMS-th piece of every head:
// its loads are then under way together, and the teams' sums are added in order.
constexpr int TEAM = HD / 4, JOIN_AT_ONCE = 8, FEW_PIECES = 8;
struct Joined {
  float4 o;
  float m, l;
  // (a part whose scores are no numbers has a maximum of -inf and passes its sum on)
  __device__ __forceinline__ void raise(float top) {
    const float mine = m == -INFINITY ? 0.f : fast_exp2(m - top);
    o.x *= mine, o.y *= mine, o.z *= mine, o.w *= mine, l *= mine, m = top;
  }
  __device__ __forceinline__ void add(float4 v, float vm, float vl) {      // of a part not above m
    const float w = (vm == -INFINITY ? 0.f : fast_exp2(vm - m)) * vl;
    o.x = fmaf(w, v.x, o.x), o.y = fmaf(w, v.y, o.y), o.z = fmaf(w, v.z, o.z), o.w = fmaf(w, v.w, o.w);
    l += w;
  }
};
template <int JOIN_THREADS>
__global__ void __launch_bounds__(JOIN_THREADS)
quant_join_kernel(const DecodeArgs a) {
  constexpr int TEAMS = JOIN_THREADS / TEAM;
  __shared__ float4 part[TEAMS][TEAM];
  __shared__ float2 part_ml[TEAMS];
  pdl_trigger();
  pdl_wait();
  const int hc = blockIdx.x / a.B, b = blockIdx.x - hc * a.B;
  const int kvh = hc / a.chunks, chunk = hc - kvh * a.chunks, G = a.nh / a.nkv;
  const int h0 = kvh * G + chunk * a.rows, nrows = min(a.rows, G - chunk * a.rows);
  const int2 info = __ldcg(a.info + blockIdx.x);
  if (info.y == 1) return;
  const int team = threadIdx.x / TEAM, c = threadIdx.x - team * TEAM;
  // the item's first piece is the second part of its block, the others are the first parts of theirs
  const size_t first = (size_t)info.x * 2 * a.rows;
  const bool few = info.y <= FEW_PIECES;
  const int start = few ? 0 : team, stride = few ? 1 : TEAMS;
  const auto store = [&](int r, float4 v, float inv) {
    const size_t at = ((size_t)b * a.nh + h0 + r) * HD + 4 * c;
    v.x *= inv, v.y *= inv, v.z *= inv, v.w *= inv;
    if (a.out_f32) {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + at) = v;
    } else {
      __nv_bfloat162* d = reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<bf16*>(a.out) + at);
      d[0] = __floats2bfloat162_rn(v.x, v.y);
      d[1] = __floats2bfloat162_rn(v.z, v.w);
    }
  };
  for (int r0 = few ? blockIdx.y * TEAMS : blockIdx.y; r0 < nrows; r0 += few ? gridDim.y * TEAMS : gridDim.y) {
    const int r = few ? r0 + team : r0;
    Joined sum = {make_float4(0.f, 0.f, 0.f, 0.f), -INFINITY, 0.f};
    if (team < TEAMS && r < nrows) {                      // (head sizes that do not divide the block)
      const float2* ml = a.pml + first + r;
      const float* po = a.po + (first + r) * HD + 4 * c;
      for (int i0 = start; i0 < info.y; i0 += JOIN_AT_ONCE * stride) {
        float2 x[JOIN_AT_ONCE];
        float4 v[JOIN_AT_ONCE];
#pragma unroll
        for (int k = 0; k < JOIN_AT_ONCE; ++k) {
          const int i = i0 + k * stride;
          x[k] = make_float2(-INFINITY, 0.f), v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i < info.y) {
            const size_t part = (size_t)(i ? 2 * i : 1) * a.rows;
            x[k] = __ldcg(ml + part);
            v[k] = __ldcg(reinterpret_cast<const float4*>(po + part * HD));
          }
        }
        float top = sum.m;
#pragma unroll
        for (int k = 0; k < JOIN_AT_ONCE; ++k) top = fmaxf(top, x[k].x);
        sum.raise(top);
#pragma unroll
        for (int k = 0; k < JOIN_AT_ONCE; ++k) sum.add(v[k], x[k].x, x[k].y);
      }
    }
    if (few) {
      if (team < TEAMS && r < nrows) store(r, sum.o, 1.f / sum.l);
      continue;
    }
    __syncthreads();                                      // (the row before has been read)
    if (team < TEAMS) part[team][c] = sum.o;
    if (team < TEAMS && c == 0) part_ml[team] = make_float2(sum.m, sum.l);
    __syncthreads();
    if (team == 0) {
      float top = part_ml[0].x;
#pragma unroll
      for (int i = 1; i < TEAMS; ++i) top = fmaxf(top, part_ml[i].x);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float l = 0.f;
#pragma unroll
      for (int i = 0; i < TEAMS; ++i) {                   // (a team's o is not divided by its sum)
        const float4 v = part[i][c];
        const float2 x = part_ml[i];
        const float w = x.x == -INFINITY ? 0.f : fast_exp2(x.x - top);
        o.x = fmaf(w, v.x, o.x), o.y = fmaf(w, v.y, o.y), o.z = fmaf(w, v.z, o.z), o.w = fmaf(w, v.w, o.w);
        l = fmaf(w, x.y, l);
      }
      store(r, o, 1.f / l);
    }
  }
}

constexpr int kTwoLaunches = -100;        // not an error: the joining kernel was launched too
template <int NT, bool FP8, typename T, bool TMA, bool STEP>
int launch_decode(DecodeArgs a, int sms, void* scratch, size_t scratch_bytes, cudaStream_t stream) {
  constexpr auto kernel = quant_decode_kernel<NT, FP8, T, TMA, STEP>;
  constexpr int results = 8 * NT * result_row(NT) * 4;
  constexpr int smem = 1024 + WARPS * (STAGES * (STAGE + SCALES) + (results <= STAGE ? 0 : results));
  static OncePerDevice once;
  static int blocks_a_sm[OncePerDevice::kMaxDevices];
  int dev = 0;
  const int rc = once.run([&]() {
    cudaGetDevice(&dev);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks_a_sm[dev], kernel, THREADS, smem);
  });
  if (rc) return rc;
  if (cudaGetDevice(&dev) != cudaSuccess) return -9;
  const int heads = a.nkv * a.chunks;
  const long long items = (long long)a.B * heads;
  const long long keys = a.span ? std::min(std::abs((long long)a.span), (long long)a.limit) : a.limit;
  const long long places = (long long)sms * std::min(std::max(1, blocks_a_sm[dev]), kMostBlocks);
  a.cluster = 1;
  if (keys > kShortKeys)
    while (a.cluster < kMostOfCluster && items * a.cluster * 2 <= places && a.cluster * kLeastTiles * TILE < keys) a.cluster *= 2;
  if (a.cluster > 1 && keys * (places - items * a.cluster) > kUnevenKeys * places * a.cluster) a.cluster = 1;
  a.stream = a.cluster == 1 && (keys > kMiddleKeys || (keys > kShortKeys && items < sms));
  const long long blocks = a.stream ? places : items * a.cluster;
  if (items > 0x7fffffffLL || blocks > 0x7fffffffLL) return -5;
  if (a.stream || a.cluster > 1) {
    const size_t rows = (size_t)blocks * 2 * a.rows, head = ((size_t)items * 8 + 15) / 16 * 16;
    if (scratch_bytes < head + rows * (HD + 2) * 4) return -7;
    a.info = (int2*)scratch;
    a.po = (float*)((char*)scratch + head);
    a.pml = (float2*)(a.po + rows * HD);
  }
  CUtensorMap map = {};
  if constexpr (TMA) {
    // a head's channels, the places of a page, a page's rows of heads (keys, then values), pages
    const EncodeTiledFn encode = encode_fn();
    const cuuint64_t dims[4] = {HD, (cuuint64_t)a.page, 2 * (cuuint64_t)a.nkv, (cuuint64_t)a.pages};
    const cuuint64_t strides[3] = {HD, (cuuint64_t)a.page * HD, 2 * (cuuint64_t)a.nkv * a.page * HD};
    const cuuint32_t box[4] = {SW, (cuuint32_t)a.unit, 2, 1}, steps[4] = {1, 1, 1, 1};
    if (!encode || encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, a.codes, dims, strides, box, steps,
                          CU_TENSOR_MAP_INTERLEAVE_NONE,
                          SW == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return -8;
  }
  const int e = launch_kernel_cluster_dims(kernel, dim3((unsigned)blocks), dim3(THREADS), smem, stream, a.cluster, true, a, map);
  if (e || !a.stream) return e;
  // few items (which have many parts): a block a head, with more teams
  const int j = items * a.rows <= 8LL * sms
                    ? launch_kernel(quant_join_kernel<512>, dim3((unsigned)items, a.rows), dim3(512), 0, stream, a)
                    : launch_kernel(quant_join_kernel<256>, dim3((unsigned)items), dim3(256), 0, stream, a);
  return j ? j : kTwoLaunches;
}

}  // namespace
}  // namespace gf

using namespace gf;

GF_DEFINE_PDL_SWITCH

// A call: q [B, nh HD], or with `step` q | k | v [B, (nh + 2 nkv) HD] and the table of angles as gf_quant_write takes
// it.  Scratch: room for two parts of an item a block, of at most kMostBlocks blocks an SM, and 8 bytes an item;
// none is needed where tables hold no more than kShortKeys keys.
struct DecodeCall {
  const void* q;
  long long q_stride, f32;
  void* codes;
  long long fp8;
  float* scales;
  const int* block_table;
  long long table_stride, table_width;
  const int* lengths;
  long long pages;
  void* out;
  long long B, nh, nkv, page, span, step;
  const float* table;
  long long table_rows, rot, neighbours, sms;
  void* scratch;
  long long scratch_bytes;
  cudaStream_t stream;
  int* err;                   // set where a copy does not come within the limit of a wait
  double scale;
};
static_assert(sizeof(DecodeCall) == 28 * 8, "the caller packs it");

// Returns 0, or kTwoLaunches, or an error.
GF_EXPORT int gf_quant_decode(const DecodeCall* call) {
  const DecodeCall& c = *call;
  if (c.B <= 0) return c.B < 0 ? -3 : 0;
  if (c.nkv < 1 || c.nh < c.nkv || c.nh % c.nkv || c.nh > 1 << 20 || c.page < 1 || c.pages < 1 || c.table_width < 0 ||
      c.B > 1 << 24 || c.sms < 1 || c.span > 0x7fffffff || c.span < -0x7fffffff)
    return -3;
  if (c.step && (c.rot < 0 || c.rot % 2 || c.rot > HD || (c.rot && (!c.table || c.table_rows < 1)))) return -3;
  if ((size_t)c.codes % 16 || (size_t)c.scales % 8) return -3;
  if (c.q_stride > 0x7fffffff || c.q_stride < 0 || c.table_stride > 0x7fffffff) return -3;
  DecodeArgs a = {};
  a.q = c.q, a.q_stride = (int)c.q_stride;
  a.codes = (uint8_t*)c.codes, a.scales = c.scales;
  a.block_table = c.block_table, a.table_stride = (int)c.table_stride;
  a.limit = (int)std::min(c.table_width * c.page, 0x7fffffe0LL - 64);
  a.pages = (int)c.pages, a.lengths = c.lengths, a.out = c.out, a.out_f32 = c.f32 != 0;
  a.B = (int)c.B, a.nh = (int)c.nh, a.nkv = (int)c.nkv, a.page = (int)c.page, a.span = (int)c.span;
  a.scale = (float)c.scale;
  a.page_shift = (a.page & (a.page - 1)) == 0 ? __builtin_ctz(a.page) : -1;
  a.table = c.table, a.table_rows = c.table_rows > 0 ? (int)c.table_rows : 1, a.rot = (int)c.rot;
  a.neighbours = c.neighbours != 0;
  a.unit = a.page % 16 ? 8 : 16, a.err = c.err;
  const int G = a.nh / a.nkv;
  a.chunks = (G + 15) / 16, a.rows = (G + a.chunks - 1) / a.chunks;
  const auto go = [&](auto nt, auto kind, auto type, auto whole, auto fused) {
    return launch_decode<decltype(nt)::value, decltype(kind)::value, decltype(type), decltype(whole)::value,
                         decltype(fused)::value>(a, (int)c.sms, c.scratch, (size_t)c.scratch_bytes, c.stream);
  };
  const auto pick_bool = [](bool x, auto next) {
    return x ? next(std::true_type()) : next(std::false_type());
  };
  return pick_bool(c.fp8 != 0, [&](auto kind) {
    // (whole copies: keys of a unit lie in one page)
    const auto pick_tma = [&](auto next) {
      if constexpr (SWIZZLED) return pick_bool(a.page % 8 == 0 && (size_t)c.scales % 16 == 0, next);
      else return next(std::false_type());
    };
    return pick_tma([&](auto whole) {
      return pick_bool(c.step != 0, [&](auto fused) {
        using One = std::integral_constant<int, 1>;
        using Two = std::integral_constant<int, 2>;
        if (c.f32) return a.rows > 8 ? go(Two(), kind, float(), whole, fused) : go(One(), kind, float(), whole, fused);
        return a.rows > 8 ? go(Two(), kind, bf16(), whole, fused) : go(One(), kind, bf16(), whole, fused);
      });
    });
  });
}
