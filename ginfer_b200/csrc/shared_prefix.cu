// Attention of a batch's newest tokens over a prefix that a group of requests shares and over their own tokens, compiled
// for one head size (-DGF_HEAD_DIM=<multiple of 16, at most 256>):
//   out[t, h] = sum_c softmax_c(scale <q[t, h], K_c>) V_c.
#ifndef GF_HEAD_DIM
#define GF_HEAD_DIM 128
#endif

#include <cstdlib>

#include "attention_tc.cuh"
#include "mma_bits.cuh"
#include "shared_prefix.cuh"

#if GF_HEAD_DIM == 64 || GF_HEAD_DIM == 128
#define GF_PREFIX_TC 1
#else
#define GF_PREFIX_TC 0
#endif

// (Internal to this library: a static of a template would be shared with the libraries of other head sizes.)
namespace gf {
namespace {

constexpr int HD = GF_HEAD_DIM;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size must be a multiple of 16, <= 256");

__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, int* err, int code) {
  const uint32_t addr = smem_u32(bar);
  for (uint32_t spin = 0; spin < kSpinLimit; ++spin) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(addr), "r"(parity) : "memory");
    if (done) return true;
    if (spin > 1024) __nanosleep(64);
  }
  if (err) atomicCAS(err, 0, code);
  return false;
}

// ------------------------------------------------------------------------------------- pieces on mma.sync
constexpr int TILE = 64;                         // keys of a tile
constexpr int MOST_ROWS = 64;                    // rows of a tile of them
constexpr int CONSUMERS = 4, THREADS = 32 * (CONSUMERS + 1);
constexpr int KCH = HD / 16;
// A tile of keys or values in shared memory: head sizes that are a multiple of 64 as TMA's 128-byte swizzle leaves them (64
// channels of 64 keys, then the next 64), others in rows of an odd number of 16-byte chunks.
constexpr bool SWIZZLED = HD % 64 == 0;
constexpr int PADDED = HD + 8;
constexpr uint32_t PLANE = SWIZZLED ? TILE * HD * 2 : TILE * PADDED * 2, STAGE = 2 * PLANE;
constexpr int STAGES = HD <= 64 ? 4 : HD <= 96 ? 3 : 2;
constexpr int BLOCKS_AN_SM = HD <= 128 ? 2 : 1;
__device__ __forceinline__ uint32_t place(int key, int ch) {       // byte offset of 8 channels of a key
  if constexpr (SWIZZLED)
    return (uint32_t)(ch >> 6) * (TILE * 128) + (uint32_t)key * 128u + (uint32_t)((((ch >> 3) & 7) ^ (key & 7)) << 4);
  else
    return (uint32_t)key * (PADDED * 2) + (uint32_t)ch * 2u;
}
constexpr int MERGE_ROW = HD + 8;                // floats from a row to the next one in the warps' exchange
constexpr uint32_t MERGE = (CONSUMERS - 1) * 16 * (MERGE_ROW + 2) * 4;
constexpr uint32_t PIECES_SMEM = STAGES * STAGE + MERGE + 2 * STAGES * 8 + 1024;

enum { OWN = 0, BOTH = 1, PREFIX = 2 };          // a request's own tokens, with its prefix, a group's prefix

struct PieceArgs {
  PrefixArgs a;
  int mode, tma, joined;       // joined: another kernel adds a row's pieces up (else every item is whole)
  int after;                   // the launch runs beside the one before it, whose results the joining kernel reads, too
  int sms;
  Shape far_shape;             // of the prefixes' kernel, where there is one: its rows, tiles and cost of a tile
  int far_tile, far_H;
  float far_cost;
  Shape shape, own_shape;      // own_shape: of own tokens
  int H;                       // kv heads * chunks (of own tokens)
  int places;                  // for pieces of prefixes
  int* chunk;                  // PREFIX: where the length of a chunk is written down
  OwnPlan* plan;
  float* far_o;                // [places][rows][HD]: pieces of prefixes
  float2* far_ml;
  float* cut_o;                // [blocks][2][MOST_ROWS][HD]: of cut items
  float2* cut_ml;
  float* row_o;                // [T][nh][HD]: of whole items, where a prefix is to be joined
  float2* row_ml;
  int* err;
};

// A part of an item: tiles [from, from + count) of prefix tiles, then own tiles.
struct Piece {
  int first, tokens, hc, from, count, far, far_len, near_len;
  int last;                    // the last own token that the first row's sees; the next token's sees one more
  const int *far_table, *near_table;
  enum { FINAL, ROW, CUT, FAR } to;
  size_t at;                   // CUT, FAR: the place
};
// The pieces of a block, one after the other; every warp goes through them by itself.
struct Pieces {
  const PieceArgs& p;
  Cursor cur;
  Request req;
  RawRequest ahead;            // the next request's numbers, on their way
  GroupTiles groups;
  int chunk, index, stride;
  __device__ __forceinline__ void start(const Cursor& c) {
    cur = c;
    if (cur.todo > 0) {
      req = request_of(p.a, cur.b, p.mode == BOTH, TILE);
      ahead.load(p.a, cur.b + 1 < p.a.B ? cur.b + 1 : 0, p.mode == BOTH);
    }
  }
  __device__ __forceinline__ void start(const GroupTiles& g, int chunk_, int blocks) {
    groups = g, chunk = chunk_, index = blockIdx.x, stride = blocks;
    if (index >= blocks) index = p.places;
  }
  __device__ __forceinline__ bool next(Piece& x) {
    const PrefixArgs& a = p.a;
    if (p.mode == PREFIX) {
      PrefixItem it;
      if (index >= p.places || !find_item(a, groups, p.H, p.shape.tokens, TILE, chunk, index, it)) return false;
      x.first = it.first, x.tokens = it.count, x.hc = it.hc;
      x.from = it.split * chunk, x.count = min(chunk, it.tiles - x.from);
      x.far = it.tiles, x.far_len = it.length, x.near_len = 0, x.last = -1;
      x.far_table = a.prefix_table + (size_t)it.g * a.prefix_stride, x.near_table = nullptr;
      x.to = Piece::FAR, x.at = index;
      index += stride;
      return true;
    }
    if (!p.joined) {
      const int done = cur.rt * p.shape.tokens;
      if (done >= req.count) return false;
      x.first = req.first + done, x.tokens = min(p.shape.tokens, req.count - done), x.hc = cur.hc;
      x.from = 0, x.count = req.tiles();
      x.far = req.far, x.far_len = req.shared, x.near_len = req.len, x.last = req.len - req.count + done;
      x.far_table = a.prefix_table + (size_t)max(req.g, 0) * a.prefix_stride;
      x.near_table = a.table + (size_t)cur.b * a.table_stride;
      x.to = Piece::FINAL;
      cur.rt += gridDim.x;
      return true;
    }
    while (cur.todo > 0) {
      const int tiles = req.tiles(), units = req.units(), done = cur.rt * p.shape.tokens, from = cur.off;
      const int count = (int)min(cur.todo, (long long)(units - from));
      const bool some = from < tiles;              // (else only the item's end, which costs time and has no tiles)
      if (some) {
        x.first = req.first + done, x.tokens = min(p.shape.tokens, req.count - done), x.hc = cur.hc;
        x.from = from, x.count = min(count, tiles - from);
        x.far = req.far, x.far_len = req.shared, x.near_len = req.len, x.last = req.len - req.count + done;
        x.far_table = a.prefix_table + (size_t)max(req.g, 0) * a.prefix_stride;
        x.near_table = a.table + (size_t)cur.b * a.table_stride;
        const bool starts = from == 0, ends = from + x.count == tiles;
        x.to = starts && ends ? (p.mode == BOTH ? Piece::FINAL : Piece::ROW) : Piece::CUT;
        x.at = (size_t)blockIdx.x * 2 + (starts ? 1 : 0);
      }
      // on to the next
      cur.todo -= count, cur.off = 0;
      if (cur.todo > 0 && ++cur.rt >= req.row_tiles(p.shape.tokens)) {
        cur.rt = 0;
        do {
          if (++cur.b == a.B) cur.b = 0, ++cur.hc;
          req = ahead.get(a, TILE);
          ahead.load(a, cur.b + 1 < a.B ? cur.b + 1 : 0, p.mode == BOTH);
        } while (req.count == 0);
      }
      if (some) return true;
    }
    return false;
  }
};
// Tile x of a piece's sequence: whose it is, its first key and the sequence's end.
struct Keys {
  const int* table;
  int key0, end;
};
__device__ __forceinline__ Keys keys_of(const Piece& x, int tile) {
  if (tile < x.far) return {x.far_table, tile * TILE, x.far_len};
  return {x.near_table, (tile - x.far) * TILE, x.near_len};
}

// One online-softmax update of a warp's 16 rows (the thread's: two) over 8 * NT keys from `key` on of the tile in `stage`;
// row i of the pair sees the keys up to seen[i].
template <int NT>
__device__ __forceinline__ void mma_step(const unsigned char* stage, int key, int key0, const uint32_t (&qf)[KCH][4],
                                         float (&o)[HD / 8][4], float (&m)[2], float (&l)[2], const int (&seen)[2],
                                         int all_see, float scale_log2, int lane) {
  static_assert(NT % 2 == 0, "");
  float s[NT][4] = {};
  const int mi = lane >> 3, r = lane & 7;
#pragma unroll
  for (int kc = 0; kc < KCH; ++kc)
#pragma unroll
    for (int n2 = 0; n2 < NT / 2; ++n2) {
      uint32_t b[4];
      ldsm_x4(b, stage + place(key + n2 * 16 + (mi >> 1) * 8 + r, kc * 16 + (mi & 1) * 8));
      mma16816(s[2 * n2], qf[kc], b[0], b[1]);
      mma16816(s[2 * n2 + 1], qf[kc], b[2], b[3]);
    }
  const bool masked = key0 + key + 8 * NT - 1 > all_see;
  float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v = s[j][e] * scale_log2;
      if (masked && key0 + key + 8 * j + 2 * (lane & 3) + (e & 1) > seen[e >> 1]) v = -INFINITY;
      s[j][e] = v;
      mx[e >> 1] = fmaxf(mx[e >> 1], v);
    }
  float corr[2], base[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
    mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
    const float top = fmaxf(m[i], mx[i]);
    base[i] = top == -INFINITY ? 0.f : top;              // (keeps -inf - -inf out of the exponent)
    corr[i] = fast_exp2(m[i] - base[i]);
    m[i] = top;
  }
  float sum[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float w = fast_exp2(s[j][e] - base[e >> 1]);
      s[j][e] = w;
      sum[e >> 1] += w;
    }
#pragma unroll
  for (int i = 0; i < 2; ++i) l[i] = l[i] * corr[i] + sum[i];
  if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) o[n][0] *= corr[0], o[n][1] *= corr[0], o[n][2] *= corr[1], o[n][3] *= corr[1];
  }
#pragma unroll
  for (int kc = 0; kc < NT / 2; ++kc) {
    // (weights are rounded to bfloat16 for the product, as everywhere in this package; their sum is not)
    uint32_t w[4];
    w[0] = pack_bf16(s[2 * kc][0], s[2 * kc][1]);
    w[1] = pack_bf16(s[2 * kc][2], s[2 * kc][3]);
    w[2] = pack_bf16(s[2 * kc + 1][0], s[2 * kc + 1][1]);
    w[3] = pack_bf16(s[2 * kc + 1][2], s[2 * kc + 1][3]);
#pragma unroll
    for (int n2 = 0; n2 < HD / 16; ++n2) {
      uint32_t b[4];
      ldsm_x4_t(b, stage + PLANE + place(key + kc * 16 + (mi & 1) * 8 + r, n2 * 16 + (mi >> 1) * 8));
      mma16816(o[2 * n2], w, b[0], b[1]);
      mma16816(o[2 * n2 + 1], w, b[2], b[3]);
    }
  }
}

__global__ void __launch_bounds__(THREADS, BLOCKS_AN_SM)
prefix_pieces_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const PieceArgs p) {
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char* ring = raw + ((0u - smem_u32(raw)) & 1023u);               // (a swizzle counts from 1 KB)
  float* merge = reinterpret_cast<float*>(ring + STAGES * STAGE);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + STAGES * STAGE + MERGE);
  uint64_t* empty = full + STAGES;
  __shared__ int chunk_s, far_s;
  __shared__ long long counts[CONSUMERS];
  __shared__ Cursor found_s;
  const PrefixArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&full[i])), "r"(32));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&empty[i])), "r"(CONSUMERS));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (!p.after) pdl_wait();
  if (p.mode == PREFIX) pdl_trigger();
  Pieces pieces{p};
  const bool both = p.mode == BOTH;
  if (p.mode == PREFIX || p.after) {
    // how the prefixes and the own tokens share the SMs, and the prefixes' chunks
    GroupTiles t{};
    FarWork f{};
    if (warp == CONSUMERS) f = far_work(a, t, p.far_H, p.far_shape.tokens, p.far_tile);
    const OwnWork w = own_work<32 * CONSUMERS>(a, p.own_shape.tokens, TILE, both, counts);
    if (warp == CONSUMERS) {
      const int share = far_share(p.sms, f.units, p.far_cost, w.total * p.H);
      if (lane == 0) far_s = share;
      if (p.mode == PREFIX) {
        const int chunk = plan_chunk(a, t, f, p.far_H, p.far_shape.tokens, p.far_tile, max(1, share * BLOCKS_AN_SM), p.places, 3);
        if (lane == 0) {
          chunk_s = chunk;
          if (blockIdx.x == 0) *p.chunk = chunk;
        }
      }
    }
    __syncthreads();
    const int far = far_s;
    if (p.mode == PREFIX) {
      if (warp != CONSUMERS) t.load(a, lane, p.shape.tokens, TILE);
      pieces.start(t, chunk_s, far * BLOCKS_AN_SM);
    } else {
      pieces.start(find_run<32 * CONSUMERS>(a, w, p.H, p.shape.tokens, TILE, both, blockIdx.x, max(p.sms - far, 1) * BLOCKS_AN_SM,
                                            blockIdx.x == 0 ? p.plan : nullptr, &found_s));
    }
  } else if (p.joined) {
    const OwnWork w = own_work<32 * CONSUMERS>(a, p.shape.tokens, TILE, both, counts);
    pieces.start(find_run<32 * CONSUMERS>(a, w, p.H, p.shape.tokens, TILE, both, blockIdx.x, gridDim.x,
                                          blockIdx.x == 0 ? p.plan : nullptr, &found_s));
  } else {
    // a block an item: (row tile, request, heads), and the row tiles behind it that the grid leaves out
    pieces.cur = {(int)blockIdx.z, (int)blockIdx.y, (int)blockIdx.x, 0, 0};
    pieces.req = request_of(a, blockIdx.y, true, TILE);
    __syncthreads();
  }
  Piece x;
  int st = 0;
  uint32_t ph = 0;
  bool ok = true;
  if (warp == CONSUMERS) {
    // ---------------------------------------------------------------- the loader
    // A tile within its sequence comes by TMA where that serves the pages, a box of a page and 64 channels; the last of a
    // sequence comes by cp.async, which leaves zeros behind its end.  A tile's places are looked up while the one before comes.
    const int box = min(a.page, TILE), boxes = TILE / box;
    auto look = [&](const Piece& y, int tile, int (&slot)[2]) {
      const Keys k = keys_of(y, tile);
#pragma unroll
      for (int u = 0; u < 2; ++u)
        slot[u] = k.end > 0 ? slot_of(a, k.table, min(k.key0 + lane + 32 * u, k.end - 1)) : 0;
    };
    int issued = 0;
    while (ok && pieces.next(x)) {
      if (x.far_len + x.near_len == 0) continue;
      const int kvh = x.hc / p.shape.chunks;
      int slot[2], ahead[2] = {0, 0};
      look(x, x.from, slot);
      for (int i = 0; i < x.count; ++i) {
        const Keys k = keys_of(x, x.from + i);
        if (i + 1 < x.count) look(x, x.from + i + 1, ahead);
        if (!wait_bar(&empty[st], ph ^ 1u, p.err, 21)) {
          ok = false;
          break;
        }
        unsigned char* stage = ring + st * STAGE;
        if (SWIZZLED && p.tma && k.key0 + TILE <= k.end) {
          // (what this warp's cp.async wrote there is out of the way of the copies)
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          if (lane == 0)
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(&full[st])), "r"(STAGE) : "memory");
          else
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&full[st])) : "memory");
          __syncwarp();
          const int ops = 2 * (HD / 64) * boxes;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int op = lane + 32 * u, bx = op % boxes, half = op / boxes % (HD / 64 ? HD / 64 : 1),
                      plane = op / (boxes * (HD / 64 ? HD / 64 : 1)), key = bx * box;
            const int s0 = __shfl_sync(0xffffffffu, slot[0], key & 31), s1 = __shfl_sync(0xffffffffu, slot[1], key & 31);
            if (op < ops)
              tma_load_2d(stage + plane * PLANE + half * (TILE * 128) + key * 128, plane ? &vmap : &kmap, &full[st],
                          kvh * HD + half * 64, key < 32 ? s0 : s1);
          }
        } else {
          constexpr int CH = HD / 8;
          const bf16* kp = static_cast<const bf16*>(a.k);
          const bf16* vp = static_cast<const bf16*>(a.v);
          const size_t stride = (size_t)a.nkv * HD;
#pragma unroll 4
          for (int j = 0; j < TILE * CH / 32; ++j) {
            const int idx = j * 32 + lane, row = idx / CH, ch = (idx - row * CH) * 8;
            const int s0 = __shfl_sync(0xffffffffu, slot[0], row & 31), s1 = __shfl_sync(0xffffffffu, slot[1], row & 31);
            const size_t off = (size_t)(row < 32 ? s0 : s1) * stride + (size_t)kvh * HD + ch;
            const bool there = k.key0 + row < k.end;
            cp_async16(stage + place(row, ch), kp + off, there);
            cp_async16(stage + PLANE + place(row, ch), vp + off, there);
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[st])) : "memory");
        }
        slot[0] = ahead[0], slot[1] = ahead[1];
        ++issued;
        if (++st == STAGES) st = 0, ph ^= 1u;
      }
    }
    // (a wait that ran out: nothing may still be on its way into this block's memory when it ends)
    if (!ok)
      for (int i = max(0, issued - STAGES); i < issued; ++i) wait_bar(&full[i % STAGES], (i / STAGES) & 1, p.err, 23);
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // ---------------------------------------------------------------- the consumers
    // 16 rows a warp.  Where there are few rows, several warps share them and take different keys of a tile; their results
    // are added up through shared memory.
    const float scale_log2 = a.scale * LOG2E;
    const int g = lane >> 2, t = lane & 3, each = a.nh / a.nkv;
    while (pieces.next(x)) {               // (behind a wait that ran out, too: the warps meet at a barrier)
      const int kvh = x.hc / p.shape.chunks, part = x.hc - kvh * p.shape.chunks;
      const int h0 = kvh * each + part * p.shape.heads, heads = min(p.shape.heads, each - part * p.shape.heads);
      const int rows = x.tokens * heads, groups = (rows + 15) >> 4;
      const int sharing = groups == 1 ? 4 : groups == 2 ? 2 : 1;
      const int mine = groups == 1 ? 0 : groups == 2 ? warp & 1 : warp, share = groups == 1 ? warp : groups == 2 ? warp >> 1 : 0;
      const bool active = mine < groups;
      int token[2], head[2], see[2];
      bool real[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = mine * 16 + g + 8 * i;
        real[i] = r < rows;
        token[i] = real[i] ? r / heads : 0;
        head[i] = h0 + (real[i] ? r - token[i] * heads : 0);
        // (rows that are none see everything, and nobody sees them)
        see[i] = real[i] ? min(x.last + token[i], x.near_len - 1) : 0x7fffffff;
        token[i] += x.first;
      }
      uint32_t qf[KCH][4];
      {
        const bf16* q0 = static_cast<const bf16*>(a.q) + (size_t)token[0] * a.q_stride + (size_t)head[0] * HD + 2 * t;
        const bf16* q1 = static_cast<const bf16*>(a.q) + (size_t)token[1] * a.q_stride + (size_t)head[1] * HD + 2 * t;
#pragma unroll
        for (int kc = 0; kc < KCH; ++kc) {
          qf[kc][0] = real[0] ? __ldcg(reinterpret_cast<const unsigned*>(q0 + kc * 16)) : 0u;
          qf[kc][1] = real[1] ? __ldcg(reinterpret_cast<const unsigned*>(q1 + kc * 16)) : 0u;
          qf[kc][2] = real[0] ? __ldcg(reinterpret_cast<const unsigned*>(q0 + kc * 16 + 8)) : 0u;
          qf[kc][3] = real[1] ? __ldcg(reinterpret_cast<const unsigned*>(q1 + kc * 16 + 8)) : 0u;
        }
      }
      // what every row of the warp sees, and what one of them does
      int all = min(see[0], see[1]), any = max(real[0] ? see[0] : -1, real[1] ? see[1] : -1);
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        all = min(all, __shfl_xor_sync(0xffffffffu, all, d));
        any = max(any, __shfl_xor_sync(0xffffffffu, any, d));
      }
      float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
      for (int n = 0; n < HD / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
      const int count = x.far_len + x.near_len > 0 ? x.count : 0;
      for (int i = 0; i < count && ok; ++i) {
        const Keys k = keys_of(x, x.from + i);
        ok = wait_bar(&full[st], ph, p.err, 22);
        if (!ok) break;
        const unsigned char* stage = ring + st * STAGE;
        const bool far = x.from + i < x.far;
        const int seen[2] = {far ? k.end - 1 : see[0], far ? k.end - 1 : see[1]};
        const int all_see = far ? k.end - 1 : all, any_sees = far ? k.end - 1 : any;
        if (active) {
          if (sharing == 4) {
            if (k.key0 + share * 16 <= any_sees)
              mma_step<2>(stage, share * 16, k.key0, qf, o, m, l, seen, all_see, scale_log2, lane);
          } else {
#pragma unroll 1
            for (int key = share * 32; key < TILE; key += 32 * sharing)
              if (k.key0 + key <= any_sees) mma_step<4>(stage, key, k.key0, qf, o, m, l, seen, all_see, scale_log2, lane);
          }
        }
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&empty[st])) : "memory");
        if (++st == STAGES) st = 0, ph ^= 1u;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      }
      if (sharing > 1) {
        // the others' results into the first one's registers
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (share > 0) {
          float* to = merge + (groups == 1 ? share - 1 : mine) * 16 * (MERGE_ROW + 2);
#pragma unroll
          for (int n = 0; n < HD / 8; ++n) {
            *reinterpret_cast<float2*>(to + g * MERGE_ROW + n * 8 + 2 * t) = make_float2(o[n][0], o[n][1]);
            *reinterpret_cast<float2*>(to + (g + 8) * MERGE_ROW + n * 8 + 2 * t) = make_float2(o[n][2], o[n][3]);
          }
          if (t == 0) {
            float2* ml = reinterpret_cast<float2*>(to + 16 * MERGE_ROW);
            ml[g] = make_float2(m[0], l[0]), ml[g + 8] = make_float2(m[1], l[1]);
          }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (share == 0) {
          for (int w = 0; w < sharing - 1; ++w) {
            const float* from = merge + (groups == 1 ? w : mine) * 16 * (MERGE_ROW + 2);
            const float2* ml = reinterpret_cast<const float2*>(from + 16 * MERGE_ROW);
            float me[2], it[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float2 y = ml[g + 8 * i];
              const float top = fmaxf(m[i], y.x), base = top == -INFINITY ? 0.f : top;
              me[i] = fast_exp2(m[i] - base), it[i] = fast_exp2(y.x - base);
              m[i] = top, l[i] = l[i] * me[i] + y.y * it[i];
            }
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) {
              const float2 y0 = *reinterpret_cast<const float2*>(from + g * MERGE_ROW + n * 8 + 2 * t);
              const float2 y1 = *reinterpret_cast<const float2*>(from + (g + 8) * MERGE_ROW + n * 8 + 2 * t);
              o[n][0] = o[n][0] * me[0] + y0.x * it[0], o[n][1] = o[n][1] * me[0] + y0.y * it[0];
              o[n][2] = o[n][2] * me[1] + y1.x * it[1], o[n][3] = o[n][3] * me[1] + y1.y * it[1];
            }
          }
        }
      }
      if (ok && active && share == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (!real[i]) continue;
          const size_t row = (size_t)token[i] * a.nh + head[i];
          if (x.to == Piece::FINAL) {
            const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];            // (no key: zeros)
            bf16* to = static_cast<bf16*>(a.out) + row * HD + 2 * t;
#pragma unroll
            for (int n = 0; n < HD / 8; ++n)
              *reinterpret_cast<uint32_t*>(to + n * 8) = pack_bf16(o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
          } else {
            const int r = mine * 16 + g + 8 * i;
            const size_t at = x.to == Piece::ROW ? row : x.at * MOST_ROWS + r;
            float* to = (x.to == Piece::ROW ? p.row_o : x.to == Piece::CUT ? p.cut_o : p.far_o) + at * HD + 2 * t;
            float2* ml = x.to == Piece::ROW ? p.row_ml : x.to == Piece::CUT ? p.cut_ml : p.far_ml;
#pragma unroll
            for (int n = 0; n < HD / 8; ++n)
              *reinterpret_cast<float2*>(to + n * 8) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
            if (t == 0) ml[at] = make_float2(m[i], l[i]);
          }
        }
      }
    }
  }
  if (p.joined && p.mode != PREFIX) {
    pdl_trigger();
    // the joining kernel waits for this launch alone: its last block ends behind the one that ran beside it
    if (p.after && blockIdx.x == gridDim.x - 1) pdl_wait();
  }
}

}  // namespace
}  // namespace gf

#if GF_PREFIX_TC
#include "shared_prefix_tc.cuh"
#endif

namespace gf {
namespace {

// ------------------------------------------------------------------------------------- joining
// A row's pieces, a warp a row: those of its prefix, then those of its own tokens, in order.
struct JoinArgs {
  PieceArgs p;
  int far_tile, far_rows;      // keys of a tile and rows of a place of the prefixes' pieces; 0: there are none
  Shape far_shape;
  int own_blocks;
};
constexpr int JOIN_WARPS = 8, JOIN_CH = (HD / 4 + 31) / 32;      // a lane has channels 4 lane, 128 + 4 lane

template <typename T>
__global__ void __launch_bounds__(32 * JOIN_WARPS) prefix_join_kernel(const JoinArgs j) {
  const PieceArgs& p = j.p;
  const PrefixArgs& a = p.a;
  const int b = blockIdx.x, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, each = a.nh / a.nkv;
  pdl_trigger();
  pdl_wait();
  const bool both = p.mode == BOTH;
  const Request r = request_of(a, b, both, TILE);
  if (r.count == 0) return;
  // where its prefix's pieces are
  int splits = 0, far_mt = 0, far_first = 0;
  long long far_base = 0;
  if (j.far_tile) {
    const int g = group_of(a, b), H = a.nkv * j.far_shape.chunks, chunk = max(fresh_index(p.chunk), 1);
    for (int g0 = 0; g0 < a.G && g0 <= g; g0 += 32) {
      GroupTiles t;
      t.load(a, g0 + lane, j.far_shape.tokens, j.far_tile);
      const int s = (t.nt + chunk - 1) / chunk;
      long long items = g0 + lane < g ? (long long)t.mt * H * s : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) items += __shfl_xor_sync(0xffffffffu, items, o);
      far_base += items;
      if (g - g0 < 32) {
        splits = __shfl_sync(0xffffffffu, s, g - g0);
        far_mt = __shfl_sync(0xffffffffu, t.mt, g - g0);
        far_first = __shfl_sync(0xffffffffu, t.first, g - g0);
      }
    }
  }
  const long long run = __ldcg(&p.plan->run), per = __ldcg(&p.plan->each), base = __ldcg(&p.plan->base[b]);
  const int tiles = r.tiles(), units = r.units();
  for (int i = blockIdx.z * JOIN_WARPS + warp; i < r.count * each; i += gridDim.z * JOIN_WARPS) {
    const int token = i / each, hh = i - token * each, t = r.first + token;
    const size_t row = (size_t)t * a.nh + kvh * each + hh;
    // its own tokens' pieces: the blocks whose runs have some of its tiles
    const int rt = token / p.shape.tokens, part = hh / p.shape.heads, heads = min(p.shape.heads, each - part * p.shape.heads);
    const int own_r = (token - rt * p.shape.tokens) * heads + hh - part * p.shape.heads;
    const long long s0 = (kvh * p.shape.chunks + part) * per + base + (long long)rt * units;
    const int k0 = (int)quotient(s0, run), k1 = (int)quotient(s0 + tiles - 1, run);
    const bool cut = k1 > k0;
    if (!cut && both) continue;                          // (the row is written already)
    const int far_part = j.far_tile ? hh / j.far_shape.heads : 0;
    const int far_heads = j.far_tile ? min(j.far_shape.heads, each - far_part * j.far_shape.heads) : 1;
    const int from = t - far_first, m = j.far_tile ? from / j.far_shape.tokens : 0;
    // (the tensor cores' tiles leave room for the heads that a chunk may have, the others for those that it has)
    const int far_r = j.far_tile ? (from - m * j.far_shape.tokens) * (j.far_rows == 128 ? j.far_shape.heads : far_heads) + hh -
                                       far_part * j.far_shape.heads : 0;
    const long long far_at = far_base + (long long)(kvh * j.far_shape.chunks + far_part) * splits * far_mt + m;
    const int own = cut ? k1 - k0 + 1 : 1, pieces = splits + own;
    auto find = [&](int k, const float*& o, const float2*& ml) {
      if (k < splits) {
        const long long item = far_at + (long long)k * far_mt;
        const bool there = m >= 0 && m < far_mt && item < p.places;
        const size_t at = there ? (size_t)item * j.far_rows + far_r : 0;
        o = p.far_o + at * HD, ml = there ? p.far_ml + at : nullptr;
      } else if (!cut) {
        o = p.row_o + row * HD, ml = p.row_ml + row;
      } else {
        const size_t at = ((size_t)(k0 + k - splits) * 2 + (k == splits ? 1 : 0)) * MOST_ROWS + own_r;
        o = p.cut_o + at * HD, ml = p.cut_ml + at;
      }
    };
    float top = -INFINITY, sum = 0.f, acc[JOIN_CH][4] = {};
    for (int k = 0; k < pieces; k += 32) {
      const float* po = nullptr;
      const float2* pml = nullptr;
      float2 ml = make_float2(-INFINITY, 0.f);
      if (k + lane < pieces) find(k + lane, po, pml);
      if (pml) ml = __ldcg(pml);
      const float best = fmaxf(top, warp_max(ml.x)), ref = best == -INFINITY ? 0.f : best;
      const float keep = fast_exp2(top - ref), w = fast_exp2(ml.x - ref);
      top = best;
      sum = sum * keep + warp_sum(ml.y * w);
#pragma unroll
      for (int c = 0; c < JOIN_CH; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[c][e] *= keep;
      const int n = min(32, pieces - k);
      // (eight pieces' values are on their way at once; what weighs nothing is not looked at)
      for (int q0 = 0; q0 < n; q0 += 8) {
        float4 y[8][JOIN_CH];
        float wq[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          wq[q] = __shfl_sync(0xffffffffu, w, (q0 + q) & 31);
          const float* from_o = (const float*)__shfl_sync(0xffffffffu, (unsigned long long)po, min(q0 + q, n - 1));
          if (q0 + q >= n) wq[q] = 0.f;
#pragma unroll
          for (int c = 0; c < JOIN_CH; ++c)
            y[q][c] = 128 * c + 4 * lane < HD ? __ldcg(reinterpret_cast<const float4*>(from_o + 128 * c + 4 * lane))
                                              : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int q = 0; q < 8; ++q)
#pragma unroll
          for (int c = 0; c < JOIN_CH; ++c)
            if (wq[q] != 0.f)
              acc[c][0] += wq[q] * y[q][c].x, acc[c][1] += wq[q] * y[q][c].y, acc[c][2] += wq[q] * y[q][c].z,
                  acc[c][3] += wq[q] * y[q][c].w;
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* out = static_cast<T*>(a.out) + row * HD;
#pragma unroll
    for (int c = 0; c < JOIN_CH; ++c)
      if (128 * c + 4 * lane < HD) {
        const float y[4] = {acc[c][0] * inv, acc[c][1] * inv, acc[c][2] * inv, acc[c][3] * inv};
        Quad<T>::store(out + 128 * c + 4 * lane, y);
      }
  }
}

// ------------------------------------------------------------------------------------- 32 bits
constexpr int kWarps = 4, kMostChannels = 256 / 32;

template <typename T>
__global__ void __launch_bounds__(32 * kWarps) prefix_simple_kernel(const PrefixArgs a) {
  __shared__ float part[kWarps][256], part_m[kWarps], part_l[kWarps];
  const int b = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = h / (a.nh / a.nkv);
  pdl_trigger();
  pdl_wait();
  const Rows rows = rows_of(a, b);
  const int g = group_of(a, b), shared = prefix_length(a, g), len = own_length(a, b);
  const T* k = static_cast<const T*>(a.k);
  const T* v = static_cast<const T*>(a.v);
  for (int i = 0; i < rows.count; ++i) {
    const size_t row = rows.first + i;
    const T* q = static_cast<const T*>(a.q) + row * a.q_stride + (size_t)h * a.hd;
    float x[kMostChannels], o[kMostChannels], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < kMostChannels; ++j) {
      x[j] = 32 * j + lane < a.hd ? to_f32(q[32 * j + lane]) * a.scale : 0.f;
      o[j] = 0.f;
    }
    const int keys = shared + max(len - rows.count + i + 1, 0);
    for (int c = warp; c < keys; c += kWarps) {
      const int* tbl = c < shared ? a.prefix_table + (size_t)g * a.prefix_stride : a.table + (size_t)b * a.table_stride;
      const int at = c < shared ? c : c - shared;
      const size_t slot = (size_t)page_in(a, fresh_index(tbl + at / a.page)) * a.page + at % a.page;
      const size_t off = (slot * a.nkv + kvh) * a.hd;
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < kMostChannels; ++j)
        if (32 * j + lane < a.hd) s = fmaf(x[j], to_f32(k[off + 32 * j + lane]), s);
      s = warp_sum(s);
      const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
      const float w = expf(s - base), keep = expf(m - base);
      m = top;
      l = l * keep + w;
#pragma unroll
      for (int j = 0; j < kMostChannels; ++j)
        if (32 * j + lane < a.hd) o[j] = o[j] * keep + w * to_f32(v[off + 32 * j + lane]);
    }
    __syncthreads();
    if (lane == 0) part_m[warp] = m, part_l[warp] = l;
#pragma unroll
    for (int j = 0; j < kMostChannels; ++j)
      if (32 * j + lane < a.hd) part[warp][32 * j + lane] = o[j];
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part_m[w]);
    const float base = top == -INFINITY ? 0.f : top;
    for (int w = 0; w < kWarps; ++w) sum += part_l[w] * expf(part_m[w] - base);
    T* out = static_cast<T*>(a.out) + (row * a.nh + h) * a.hd;
    for (int d = threadIdx.x; d < a.hd; d += 32 * kWarps) {
      float y = 0.f;
      for (int w = 0; w < kWarps; ++w) y += part[w][d] * expf(part_m[w] - base);
      out[d] = from_f32<T>(keys > 0 ? y / sum : 0.f);
    }
  }
}

// ------------------------------------------------------------------------------------- host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* at = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &at, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = (EncodeTiledFn)at;
  }
  return fn;
}
// 64 channels of `rows` tokens of a plane of the cache, 128-byte swizzle
bool page_map(CUtensorMap* map, const void* plane, const PrefixArgs& a, int rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)a.nkv * HD, (cuuint64_t)a.pages * a.page};
  cuuint64_t strides[1] = {(cuuint64_t)a.nkv * HD * 2};
  cuuint32_t box[2] = {64u, (cuuint32_t)rows}, steps[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(plane), dims, strides, box, steps,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

#if GF_PREFIX_TC
// 64 channels of the query heads of some rows
bool query_map(CUtensorMap* map, const PrefixArgs& a, const Shape& shape) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {(cuuint64_t)HD, (cuuint64_t)a.nh, (cuuint64_t)a.T};
  cuuint64_t strides[2] = {(cuuint64_t)HD * 2, (cuuint64_t)a.q_stride * 2};
  cuuint32_t box[3] = {64u, (cuuint32_t)shape.heads, (cuuint32_t)shape.tokens}, steps[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a.q), dims, strides, box, steps,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
#endif

}  // namespace
}  // namespace gf

using namespace gf;

GF_DEFINE_PDL_SWITCH

// What a tile of a prefix costs beside a tile of own tokens (64 keys that come from memory): 128 keys on the tensor cores with up to
// 128 rows, 64 keys on mma.sync with up to 64 rows.
constexpr float kTensorCost = 2.f, kPlainCost = 2.f;

// `words`: q, its row stride and type, k, v, pages, page, prefix_table and its stride, prefix_lens, groups, prefix limit,
// table and its stride, lengths, requests, limit, cu_groups, cu, out, rows, heads, kv heads, SMs, the rows that a request has
// at most (a hint), scratch and its bytes, err, stream; then the scale as a double.
struct Call {
  PieceArgs p;
  JoinArgs j;
  int type, blocks, longest, sms;
  bool shared, tensor;         // tensor: prefixes on the 5th-generation tensor cores
  char* scratch;
  long long room, need;
  cudaStream_t stream;

  explicit Call(const char* words) : p{}, j{} {
    const long long* w = reinterpret_cast<const long long*>(words);
    PrefixArgs& a = p.a;
    int i = 0;
    auto ptr = [&] { return reinterpret_cast<void*>(w[i++]); };
    auto num = [&] { return (int)w[i++]; };
    a.q = ptr(), a.q_stride = num(), type = num();
    a.k = ptr(), a.v = ptr(), a.pages = num(), a.page = num();
    a.prefix_table = (const int*)ptr(), a.prefix_stride = num(), a.prefix_lens = (const int*)ptr();
    a.G = num(), a.prefix_limit = num();
    a.table = (const int*)ptr(), a.table_stride = num(), a.lengths = (const int*)ptr(), a.B = num(), a.limit = num();
    a.cu_groups = (const int*)ptr(), a.cu = (const int*)ptr(), a.out = ptr();
    a.T = num(), a.nh = num(), a.nkv = num();
    sms = num();
    longest = num();
    scratch = (char*)ptr(), room = w[i++];
    p.err = (int*)ptr(), stream = (cudaStream_t)ptr();
    a.scale = (float)*reinterpret_cast<const double*>(w + i);
    a.hd = HD;
    a.page_shift = (a.page & (a.page - 1)) == 0 ? 31 - __builtin_clz(a.page) : -1;
    const char* env2 = getenv("GF_UNSHARED");
    shared = a.G > 0 && a.prefix_limit > 0 && a.T > (env2 ? atoi(env2) : 2);
    p.shape = row_shape_of(a.nh, a.nkv, MOST_ROWS);
    p.H = a.nkv * p.shape.chunks;
    p.own_shape = p.shape, p.sms = sms;
    blocks = sms * BLOCKS_AN_SM;
    // the scratch: the division, pieces of cut items, of rows, of prefixes
    need = 0;
    auto take = [&](long long bytes) {
      char* here = scratch + need;
      need += (bytes + 255) / 256 * 256;
      return here;
    };
    const long long rows = (long long)a.T * a.nh, cut = (long long)blocks * 2 * MOST_ROWS;
    p.chunk = (int*)take(4);
    p.plan = (OwnPlan*)take(16 + 8ll * a.B);
    p.cut_o = (float*)take(cut * HD * 4), p.cut_ml = (float2*)take(cut * 8);
    if (shared) {
      p.row_o = (float*)take(rows * HD * 4), p.row_ml = (float2*)take(rows * 8);
      tensor = GF_PREFIX_TC && type == GF_BF16 && a.page % 8 == 0 && 128 % a.page == 0;
      j.far_tile = tensor ? 128 : TILE, j.far_rows = tensor ? 128 : MOST_ROWS;
      j.far_shape = row_shape_of(a.nh, a.nkv, j.far_rows);
      p.far_shape = j.far_shape, p.far_tile = j.far_tile, p.far_H = a.nkv * j.far_shape.chunks;
      p.far_cost = tensor ? kTensorCost : kPlainCost;
      const long long tiles = (long long)a.nkv * j.far_shape.chunks * ((a.T + j.far_shape.tokens - 1) / j.far_shape.tokens + a.G);
      const long long least = 2ll * (tensor ? sms : blocks);
      p.places = (int)(tiles > least ? tiles : least);
      p.far_o = (float*)take((long long)p.places * j.far_rows * HD * 4);
      p.far_ml = (float2*)take((long long)p.places * j.far_rows * 8);
    }
  }
};

// The bytes of scratch that a call wants.
GF_EXPORT long long gf_prefix_scratch(const char* words) { return Call(words).need; }

GF_EXPORT int gf_prefix_attend(const char* words) {
  Call c(words);
  PieceArgs& p = c.p;
  PrefixArgs& a = p.a;
  if (a.B <= 0 || a.T <= 0) return 0;
  if (c.type != GF_BF16)
    return launch_kernel(prefix_simple_kernel<float>, dim3(a.B, a.nh), dim3(32 * kWarps), 0, c.stream, a);
  if (c.need > c.room) return -5;
  static OncePerDevice attrs;
  if (int rc = attrs.run([&] {
        return cudaFuncSetAttribute(prefix_pieces_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PIECES_SMEM);
      }))
    return rc;
  CUtensorMap mk{}, mv{};
  p.tma = SWIZZLED && a.page % 8 == 0 && (TILE % a.page == 0 || a.page % TILE == 0) && !((uintptr_t)a.k & 15) &&
          !((uintptr_t)a.v & 15);
  if (p.tma) {
    const int rows = a.page < TILE ? a.page : TILE;
    if (!page_map(&mk, a.k, a, rows) || !page_map(&mv, a.v, a, rows)) return -7;
  }
  JoinArgs& j = c.j;
  const char* env = getenv("GF_SHORT");
  if (a.prefix_limit + a.limit <= (env ? atoi(env) : 512) && a.B <= 65535 && p.H <= 65535) {
    p.mode = BOTH, p.joined = 0;
    const int row_tiles = (c.longest + p.shape.tokens - 1) / p.shape.tokens;
    return launch_kernel(prefix_pieces_kernel, dim3(row_tiles > 1 ? row_tiles : 1, a.B, p.H), dim3(THREADS), PIECES_SMEM, c.stream,
                         mk, mv, p);
  }
  if (c.shared) {
    int rc;
#if GF_PREFIX_TC
    if (c.tensor) {
      static OncePerDevice tc_attrs;
      rc = tc_attrs.run([&] {
        return cudaFuncSetAttribute(tc::prefix_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)tc::SMEM);
      });
      if (rc) return rc;
      const tc::Args t{a, j.far_shape, p.shape, p.far_H, p.H, p.places, a.pages * a.page, c.sms, TILE, p.far_cost, p.chunk, p.far_o, p.far_ml, p.err};
      CUtensorMap tq, tk, tv;
      if (!query_map(&tq, a, j.far_shape) || !page_map(&tk, a.k, a, a.page) || !page_map(&tv, a.v, a, a.page)) return -7;
      rc = launch_kernel(tc::prefix_tc_kernel, dim3(c.sms), dim3(tc::NTHREADS_TC), tc::SMEM, c.stream, tq, tk, tv, t);
    } else
#endif
    {
      p.mode = PREFIX;
      rc = launch_kernel(prefix_pieces_kernel, dim3(c.blocks), dim3(THREADS), PIECES_SMEM, c.stream, mk, mv, p);
    }
    if (rc) return rc;
    p.after = 1;
  }
  p.mode = c.shared ? OWN : BOTH, p.joined = 1;
  const int rc = launch_kernel(prefix_pieces_kernel, dim3(c.blocks), dim3(THREADS), PIECES_SMEM, c.stream, mk, mv, p);
  if (rc) return rc;
  j.p = p, j.own_blocks = c.blocks;
  // (a warp a row where the requests have as many as is said)
  const long long per = (long long)(c.longest < 1 ? 1 : c.longest) * (a.nh / a.nkv);
  const unsigned z = (unsigned)(per > 64 * JOIN_WARPS ? 64 : (per + JOIN_WARPS - 1) / JOIN_WARPS);
  return launch_kernel(prefix_join_kernel<bf16>, dim3(a.B, a.nkv, z), dim3(32 * JOIN_WARPS), 0, c.stream, j);
}
