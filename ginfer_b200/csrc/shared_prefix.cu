// Attention of a batch's newest tokens over a prefix that a group of requests shares and over their own tokens, compiled
// for one head size (-DGF_HEAD_DIM=<multiple of 16, at most 256>):
//   out[t, h] = sum_c softmax_c(scale <q[t, h], K_c>) V_c.
#ifndef GF_HEAD_DIM
#define GF_HEAD_DIM 128
#endif

#include <climits>

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
// Prefixes where the tensor cores' own kernel does not serve (heads other than 64 and 128, pages that are not multiples of 8 up
// to 128): a loading warp and four that share a tile's keys, 16 rows of q a product, up to 64 a block.  18 us for 24
// requests behind prompts of 3,001 and 1,331 tokens, 16 heads on 4 of 96, beside their own tokens, most of it starts (0.4 GFLOP).
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

struct FarArgs {
  PrefixArgs a;
  int tma;
  Shape shape, own_shape;      // rows of this kernel's tiles, of the one's that works on own tokens beside it
  int H, own_H, places, sms, own_tile;
  float cost;                  // of a tile beside one of own tokens
  FarPlan* far_plan;           // [G]
  float* far_o;                // [places][MOST_ROWS][HD]
  float2* far_ml;
  int* err;
};

// One online-softmax update of a warp's 16 rows (the thread's: two) over 8 * NT keys from `key` on of the tile in `stage`, whose first
// is key0; `last`: the sequence's last key.
template <int NT>
__device__ __forceinline__ void mma_step(const unsigned char* stage, int key, int key0, int last, const uint32_t (&qf)[KCH][4],
                                         float (&o)[HD / 8][4], float (&m)[2], float (&l)[2], float scale_log2, int lane) {
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
  const bool masked = key0 + key + 8 * NT - 1 > last;
  float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v = s[j][e] * scale_log2;
      if (masked && key0 + key + 8 * j + 2 * (lane & 3) + (e & 1) > last) v = -INFINITY;
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
  // (weights are rounded to bfloat16 for the product, as everywhere in this package; what is summed are the rounded ones: a row
  // that one key takes nearly all of gets its value as it is)
  float sum[2] = {0.f, 0.f};
  uint32_t w[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[j][i] = pack_bf16(fast_exp2(s[j][2 * i] - base[i]), fast_exp2(s[j][2 * i + 1] - base[i]));
      sum[i] += __uint_as_float(w[j][i] << 16) + __uint_as_float(w[j][i] & 0xffff0000u);
    }
#pragma unroll
  for (int i = 0; i < 2; ++i) l[i] = l[i] * corr[i] + sum[i];
  if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) o[n][0] *= corr[0], o[n][1] *= corr[0], o[n][2] *= corr[1], o[n][3] *= corr[1];
  }
#pragma unroll
  for (int kc = 0; kc < NT / 2; ++kc) {
    const uint32_t x[4] = {w[2 * kc][0], w[2 * kc][1], w[2 * kc + 1][0], w[2 * kc + 1][1]};
#pragma unroll
    for (int n2 = 0; n2 < HD / 16; ++n2) {
      uint32_t b[4];
      ldsm_x4_t(b, stage + PLANE + place(key + kc * 16 + (mi & 1) * 8 + r, n2 * 16 + (mi >> 1) * 8));
      mma16816(o[2 * n2], x, b[0], b[1]);
      mma16816(o[2 * n2 + 1], x, b[2], b[3]);
    }
  }
}

__global__ void __launch_bounds__(THREADS, BLOCKS_AN_SM)
prefix_pieces_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const FarArgs p) {
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char* ring = raw + ((0u - smem_u32(raw)) & 1023u);               // (a swizzle counts from 1 KB)
  float* merge = reinterpret_cast<float*>(ring + STAGES * STAGE);
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + STAGES * STAGE + MERGE);
  uint64_t* empty = full + STAGES;
  __shared__ int chunk_s, workers_s;
  __shared__ long long counts[CONSUMERS];
  __shared__ GroupTiles groups_s[32];
  const PrefixArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&full[i])), "r"(32));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&empty[i])), "r"(CONSUMERS));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_wait();
  pdl_trigger();               // (behind the wait: the kernel beside this one reads what was waited for)
  {
    // how the prefixes and the own tokens share the SMs, and the prefixes' chunks
    GroupTiles t{};
    FarWork f{};
    if (warp == CONSUMERS) f = far_work(a, t, p.H, p.shape.tokens, TILE);
    const OwnWork w = own_work<32 * CONSUMERS>(a, p.own_shape.tokens, p.own_tile, false, counts);
    if (warp == CONSUMERS) {
      const int workers = far_share(p.sms, f.priced, p.cost, w.total * p.own_H) * BLOCKS_AN_SM;
      const int chunk = plan_chunk(a, t, f, p.H, p.shape.tokens, TILE, max(workers, 1), p.places, 3);
      groups_s[lane] = t;
      if (lane == 0) chunk_s = chunk, workers_s = workers;
      if (blockIdx.x == 0) write_far_plan(a, t, p.H, p.shape.tokens, TILE, chunk, p.far_plan);
    }
    __syncthreads();
  }
  const int chunk = chunk_s, workers = workers_s;
  const GroupTiles groups = groups_s[lane];
  PrefixItem it;
  // the block's n-th item; by whole warps
  auto item_of = [&](int n) {
    const int index = n * workers + (int)blockIdx.x;
    return (int)blockIdx.x < workers && index < p.places && find_item(a, groups, p.H, p.shape.tokens, TILE, chunk, index, it);
  };
  int st = 0;
  uint32_t ph = 0;
  bool ok = true;
  if (warp == CONSUMERS) {
    // ---------------------------------------------------------------- the loader
    // A tile within its sequence comes by TMA where that serves the pages, a box of a page and 64 channels; the last of a
    // sequence comes by cp.async, which leaves zeros behind its end.  A tile's places are looked up while the one before comes.
    const int box = min(a.page, TILE), boxes = TILE / box;
    int issued = 0;
    for (int n = 0; ok && item_of(n); ++n) {
      const int kvh = it.hc / p.shape.chunks, from = it.split * chunk, count = min(chunk, it.tiles - from), end = it.length;
      const int* tbl = a.prefix_table + (size_t)it.g * a.prefix_stride;
      auto look = [&](int tile, int (&slot)[2]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) slot[u] = slot_of(a, tbl, min(tile * TILE + lane + 32 * u, end - 1));
      };
      int slot[2], ahead[2] = {0, 0};
      look(from, slot);
      for (int i = 0; i < count; ++i) {
        const int key0 = (from + i) * TILE;
        if (i + 1 < count) look(from + i + 1, ahead);
        // (the warp's verdict: a lane that left by itself would leave the others at the exchanges that follow)
        if (!__all_sync(0xffffffffu, wait_bar(&empty[st], ph ^ 1u, p.err, 21))) {
          ok = false;
          break;
        }
        unsigned char* stage = ring + st * STAGE;
        if (SWIZZLED && p.tma && key0 + TILE <= end) {
          // (what this warp's cp.async wrote there is out of the way of the copies)
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          if (lane == 0)
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(&full[st])), "r"(STAGE) : "memory");
          else
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&full[st])) : "memory");
          __syncwarp();
          constexpr int HALVES = HD / 64 ? HD / 64 : 1;
          const int ops = 2 * HALVES * boxes;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int op = lane + 32 * u, bx = op % boxes, half = op / boxes % HALVES, plane = op / (boxes * HALVES), key = bx * box;
            const int s0 = __shfl_sync(0xffffffffu, slot[0], key & 31), s1 = __shfl_sync(0xffffffffu, slot[1], key & 31);
            if (op < ops)
              tma_load_2d(stage + plane * PLANE + half * (TILE * 128) + key * 128, plane ? &vmap : &kmap, &full[st],
                          kvh * HD + half * 64, key < 32 ? s0 : s1);
          }
        } else {
          constexpr int CH = HD / 8;
          const bf16* kp = static_cast<const bf16*>(a.k) + (size_t)kvh * HD;
          const bf16* vp = static_cast<const bf16*>(a.v) + (size_t)kvh * HD;
          const size_t stride = (size_t)a.nkv * HD;
#pragma unroll 4
          for (int j = 0; j < TILE * CH / 32; ++j) {
            const int idx = j * 32 + lane, row = idx / CH, ch = (idx - row * CH) * 8;
            const int s0 = __shfl_sync(0xffffffffu, slot[0], row & 31), s1 = __shfl_sync(0xffffffffu, slot[1], row & 31);
            const size_t off = (size_t)(row < 32 ? s0 : s1) * stride + ch;
            const bool there = key0 + row < end;
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
    for (int n = 0; item_of(n); ++n) {     // (behind a wait that ran out, too: the warps meet at a barrier)
      const int kvh = it.hc / p.shape.chunks, part = it.hc - kvh * p.shape.chunks;
      const int h0 = kvh * each + part * p.shape.heads, heads = min(p.shape.heads, each - part * p.shape.heads);
      const int rows = it.count * heads, groups16 = (rows + 15) >> 4, from = it.split * chunk, count = min(chunk, it.tiles - from);
      const int sharing = groups16 == 1 ? 4 : groups16 == 2 ? 2 : 1;
      const int mine = groups16 == 1 ? 0 : groups16 == 2 ? warp & 1 : warp;
      const int share = groups16 == 1 ? warp : groups16 == 2 ? warp >> 1 : 0;
      const bool active = mine < groups16;
      bool real[2];
      uint32_t qf[KCH][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = mine * 16 + g + 8 * i;
        real[i] = r < rows;
        const int token = real[i] ? r / heads : 0, head = real[i] ? r - token * heads : 0;
        const bf16* q = static_cast<const bf16*>(a.q) + (size_t)(it.first + token) * a.q_stride + (size_t)(h0 + head) * HD + 2 * t;
#pragma unroll
        for (int kc = 0; kc < KCH; ++kc) {
          qf[kc][i] = real[i] ? __ldcg(reinterpret_cast<const unsigned*>(q + kc * 16)) : 0u;
          qf[kc][2 + i] = real[i] ? __ldcg(reinterpret_cast<const unsigned*>(q + kc * 16 + 8)) : 0u;
        }
      }
      float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
      for (int i = 0; i < count && ok; ++i) {
        const int key0 = (from + i) * TILE, end = it.length - 1;
        ok = __all_sync(0xffffffffu, wait_bar(&full[st], ph, p.err, 22));
        if (!ok) break;
        const unsigned char* stage = ring + st * STAGE;
        if (active) {
          if (sharing == 4) {
            if (key0 + share * 16 <= end) mma_step<2>(stage, share * 16, key0, end, qf, o, m, l, scale_log2, lane);
          } else {
#pragma unroll 1
            for (int key = share * 32; key < TILE; key += 32 * sharing)
              if (key0 + key <= end) mma_step<4>(stage, key, key0, end, qf, o, m, l, scale_log2, lane);
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
        __syncwarp();            // (the barrier wants a warp as one)
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (share > 0) {
          float* to = merge + (groups16 == 1 ? share - 1 : mine) * 16 * (MERGE_ROW + 2);
#pragma unroll
          for (int c = 0; c < HD / 8; ++c) {
            *reinterpret_cast<float2*>(to + g * MERGE_ROW + c * 8 + 2 * t) = make_float2(o[c][0], o[c][1]);
            *reinterpret_cast<float2*>(to + (g + 8) * MERGE_ROW + c * 8 + 2 * t) = make_float2(o[c][2], o[c][3]);
          }
          if (t == 0) {
            float2* ml = reinterpret_cast<float2*>(to + 16 * MERGE_ROW);
            ml[g] = make_float2(m[0], l[0]), ml[g + 8] = make_float2(m[1], l[1]);
          }
        }
        __syncwarp();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (share == 0) {
          for (int w = 0; w < sharing - 1; ++w) {
            const float* other = merge + (groups16 == 1 ? w : mine) * 16 * (MERGE_ROW + 2);
            const float2* ml = reinterpret_cast<const float2*>(other + 16 * MERGE_ROW);
            float me[2], its[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float2 y = ml[g + 8 * i];
              const float top = fmaxf(m[i], y.x), base = top == -INFINITY ? 0.f : top;
              me[i] = fast_exp2(m[i] - base), its[i] = fast_exp2(y.x - base);
              m[i] = top, l[i] = l[i] * me[i] + y.y * its[i];
            }
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) {
              const float2 y0 = *reinterpret_cast<const float2*>(other + g * MERGE_ROW + c * 8 + 2 * t);
              const float2 y1 = *reinterpret_cast<const float2*>(other + (g + 8) * MERGE_ROW + c * 8 + 2 * t);
              o[c][0] = o[c][0] * me[0] + y0.x * its[0], o[c][1] = o[c][1] * me[0] + y0.y * its[0];
              o[c][2] = o[c][2] * me[1] + y1.x * its[1], o[c][3] = o[c][3] * me[1] + y1.y * its[1];
            }
          }
        }
      }
      if (ok && active && share == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (!real[i]) continue;
          const size_t at = (size_t)(n * workers + (int)blockIdx.x) * MOST_ROWS + mine * 16 + g + 8 * i;
          float* to = p.far_o + at * HD + 2 * t;
#pragma unroll
          for (int c = 0; c < HD / 8; ++c) *reinterpret_cast<float2*>(to + c * 8) = make_float2(o[c][2 * i], o[c][2 * i + 1]);
          if (t == 0) p.far_ml[at] = make_float2(m[i], l[i]);
        }
      }
    }
  }
}

}  // namespace
}  // namespace gf

#include "shared_prefix_own.cuh"
#if GF_PREFIX_TC
#include "shared_prefix_tc.cuh"
#endif

namespace gf {
namespace {

// ------------------------------------------------------------------------------------- joining
// A row's pieces, a warp a row: those of its prefix, then those of its own tokens, in order.  Latency bounds it: the plans, then
// up to 24 pieces a row (64 from warps), 8 loads under way; 10 us by itself for 1,792 rows, 4 to 7 behind the kernels before it.
struct JoinArgs {
  own::Args p;
  int far_rows, places;        // rows of a place of the prefixes' pieces (0: there are none), places
  const FarPlan* far_plan;
  const float* far_o;
  const float2* far_ml;
};
constexpr int JOIN_WARPS = 8, JOIN_CH = (HD / 4 + 31) / 32;      // a lane has channels 4 lane, 128 + 4 lane

template <typename T>
__global__ void __launch_bounds__(32 * JOIN_WARPS, HD <= 128 ? 4 : 3) prefix_join_kernel(const JoinArgs j) {
  const own::Args& p = j.p;
  const PrefixArgs& a = p.a;
  const Shape& far_shape = p.far_shape;
  const int b = blockIdx.x, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, each = a.nh / a.nkv;
  pdl_trigger();
  pdl_wait();
  const bool both = p.both;
  const OwnPlan::Entry& e = p.plan->of[b];
  const int2 rows = __ldcg(reinterpret_cast<const int2*>(&e.first)), more = __ldcg(reinterpret_cast<const int2*>(&e.tiles));
  const long long run = __ldcg(&p.plan->run), per = __ldcg(&p.plan->each), base = __ldcg(&e.base);
  const int first = rows.x, count = rows.y, tiles = more.x, units = tiles + kItemTiles;
  if (count == 0) return;
  // where its prefix's pieces are
  int4 far{};
  if (j.far_rows && more.y >= 0) far = __ldcg(reinterpret_cast<const int4*>(j.far_plan + more.y));
  const int far_base = far.x, splits = far.y, far_mt = far.z, far_first = far.w;
  for (int i = blockIdx.z * JOIN_WARPS + warp; i < count * each; i += gridDim.z * JOIN_WARPS) {
    const int token = i / each, hh = i - token * each, t = first + token;
    const size_t row = (size_t)t * a.nh + kvh * each + hh;
    // its own tokens' pieces: the blocks whose runs have some of its tiles
    const int rt = token / p.shape.tokens, part = hh / p.shape.heads, heads = min(p.shape.heads, each - part * p.shape.heads);
    const int own_r = (token - rt * p.shape.tokens) * heads + hh - part * p.shape.heads;
    const long long s0 = (kvh * p.shape.chunks + part) * per + base + (long long)rt * units;
    const int k0 = (int)quotient(s0, run), k1 = (int)quotient(s0 + tiles - 1, run);
    const bool cut = k1 > k0;
    if (!cut && both) continue;                          // (the row is written already)
    const int far_part = j.far_rows ? hh / far_shape.heads : 0;
    const int far_heads = j.far_rows ? min(far_shape.heads, each - far_part * far_shape.heads) : 1;
    // (starts that do not rise may put a row in front of its group's first: it has no piece there)
    const int from = t - far_first, m = !j.far_rows ? 0 : from < 0 ? -1 : from / far_shape.tokens;
    // (the tensor cores' tiles leave room for the heads that a chunk may have, the others for those that it has)
    const int far_r = j.far_rows ? (from - m * far_shape.tokens) * (j.far_rows == 128 ? far_shape.heads : far_heads) + hh -
                                       far_part * far_shape.heads : 0;
    const long long far_at = (long long)far_base + (long long)(kvh * far_shape.chunks + far_part) * splits * far_mt + m;
    const int own = cut ? k1 - k0 + 1 : 1, pieces = splits + own;
    auto find = [&](int k, const float*& o, const float2*& ml) {
      if (k < splits) {
        const long long item = far_at + (long long)k * far_mt;
        const bool there = m >= 0 && m < far_mt && item < j.places;
        const size_t at = there ? (size_t)item * j.far_rows + far_r : 0;
        o = j.far_o + at * HD, ml = there ? j.far_ml + at : nullptr;
      } else if (!cut) {
        o = p.row_o + row * HD, ml = p.row_ml + row;
      } else {
        const size_t at = ((size_t)(k0 + k - splits) * 2 + (k == splits ? 1 : 0)) * p.rows + own_r;
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

// Which way a call goes, by its sizes alone (the tables' widths, not the lengths in them).
//
// Direct: an item (request, kv head) is a block's, or a cluster's of 2, 4 or 8 blocks while there are SMs for twice as many and a
// block has more than kBlockKeys bytes of the item's keys, a single one twice that (clusters of 8 find places for three quarters of the SMs: one more had
// to wait for another's end); its warps share the keys of prefix and own tokens; one launch.  Where a block has at most
// kDirectKeys, in a cluster (but for 32-bit heads above 64) twice as many, requests read at most kDirectBytes of prefixes, and the items
// are at most kDirectWaves blocks an SM: behind one another, they pay their starts.
// Direct / equal runs and their join, us: 28 heads on 4 of 128, 64 requests of 1,000 tokens (a block) 26.5 / 27.3, of 2,000 42.0 /
// 41.3; 16 of 2,500 (2 blocks) 17.2 / 23.6; 8 of 4,100 (4) 16 / 25; one of 4,000 (8) 11.0 / 20.2, of 16,000 23.7 / 31.1; 14 on 2 of
// 64, 32 of 5,000 (2) 16.9 / 24.9, one of 4,000 (8) 8.1 / 19.9; that in fp32 14.9 / 30.1, 12 of up to 2,600 (2) 27.0 / 30.9; fp32, 28 on
// 4 of 128, one of 4,000 (256 KB a block) 29.7 / 35.2, of 16,000 110 / 52.  Blocks of 128 KB, 64 KB, 32 KB: 28 on 4 of 128, one of 1,000 10.6,
// 8.8, 8.1, one of 500 9.1, 8.5, 7.7; 14 on 2 of 64, 2 of 340 one block 6.2, two 6.7; in fp32, one of 1,000 14.4, 10.6, 8.7.
// Waves: 28 on 4 of 128, 64 requests of up to 400 (1.7) 16.5 / 20.8, 96 (2.6) 23.1 / 21.1, 128 of 110 (3.5) 22.2 / 20.8, 256 of 300 (6.9) 48.8 / 33.4; 40 on
// 8, 32 of 400 (1.7) 15.8 / 20.4, 64 (3.5) 28.5 / 22.6, 512 of 150 (28) 160 / 64; 14 on 2 of 64, 128 of 600 (1.7) 14.0 / 20.5, 256 of 110 (3.5) 19.7 / 19.5, 512
// of 150 (6.9) 34.9 / 24.1; that in fp32, 128 of 400 22.9 / 29.7, 256 of 110 25.4 / 28.1, of 400 42.3 / 36.6.
constexpr long long kDirectKeys = 256 << 10, kDirectBytes = 128 << 20, kBlockKeys = 32 << 10, kDirectWaves = 2;
// Unshared: every request reads its prefix itself (from L2 but for the first), in equal runs; 2 launches instead of 3.  Where
// that is at most so many bytes, the fewer the longer a prefix is: a long one keeps warps busy that have one request's chain of
// keys to go through.  Unshared / shared, us: 28 on 4 of 128, 64 requests behind 400 tokens (52 MB) 27.5 / 31.6, 700 (92 MB) 31.5 / 32.5,
// 1,000 (131 MB) 35.6 / 33.6, 2,000 (262 MB) 51.1 / 37.0; 128 behind 400 (105 MB) 36.0 / 41.9, 700 (184 MB) 44.2 / 38.6; 16 behind 4,000 (131 MB)
// 33.5 / 30.9; 4 behind 8,000 (66 MB) 28.8 / 30.5, 6 (98 MB) 30.8 / 29.4; 2 behind 16,000 (66 MB) 35.1 / 29.4; 14 on 2 of 64, 64 behind 2,000 (66 MB)
// 22.5 / 26.9, 128 (131 MB) 34.0 / 32.1; 16 on 4 of 96, 64 behind 400 (39 MB) 30.2 / 44.6, 1,000 (98 MB) 40.3 / 44.9, 2,000 (197 MB) 59.7 / 53.1, 6 behind
// 16,000 (147 MB) 47.0 / 42.5; 8 on 4 of 256, 64 behind 400 (105 MB) 43.8 / 42.8, 700 (184 MB) 53.1 / 40.5.  fp32, 14 on 2 of 64: 64 behind 1,000 (66 MB)
// 34.3 / 37.6, 2,000 (131 MB) 48.4 / 48.6; 128 behind 1,000 (131 MB) 50.6 / 54.1, 2,000 (262 MB) 76.4 / 75.2, 4,000 (524 MB) 130 / 117.  Of 601 drawn calls
// the way that this takes is 1.4 % slower than the better one in the mean.  In 32 bits with heads above 64 registers leave 8 rows a tile, with or
// without groups: 28 on 4 of 128, 128 of 4,000, 543 unshared, 785 shared; so not at all there.
constexpr long long kUnsharedBytes = 144 << 20, kUnsharedToken = 8 << 10, kUnsharedLeast = 16 << 20;
// What a tile of a prefix costs beside a tile of own tokens (which come from memory), for the SMs' shares: 128 keys on the tensor
// cores with up to 128 rows, 64 keys on mma.sync with up to 64 rows, 16 keys in 32 bits.  Own tokens' tiles are 16 keys, 32 for heads
// of up to 64.  (kFarOver is what an item costs beside its tiles.)  us at (costs):
//  * tensor cores, 128 (7, 8, 9, 10): 28 heads on 4, 64 requests behind 8,192 tokens with up to 1,024 of their own 41.5 / 40.9 / 41.0 / 41.4,
//    128 behind 4,096, 4,096 160 / 125 / 125 / 126, 256 behind 2,048, 300 70 / 55 / 55 / 56; 40 on 8, 256 behind 32,768, 512 334 / 304 / 300 / 308,
//    128 behind 4,096, 4,096 247 / 244 / 238 / 233; 12 on 2, 32 of up to 5 rows behind 4,099, 2,048 38.7 / 38.8 / 37.6 / 39.0.  64 (5, 6, 7, 8), 14 on 2: the
//    first 28.9 / 29.8 / 29.8 / 29.4, the second 53.8 / 47.8 / 48.5 / 53.7, the third 40.0 / 32.7 / 31.5 / 31.7, 256 behind 32,768, 512 108 / 99 / 98 / 95.
//  * mma.sync, up to 128 (2.5, 3, 3.5, 4): 16 on 4 of 96, 24 of up to 3 rows behind two prompts of up to 3,001, 700 30.0 / 30.2 / 30.1 / 31.2, 128 behind
//    4,096, 2,048 162 / 133 / 127 / 133, 64 behind 8,192, 1,024 63.4 / 62.1 / 66.6 / 65.0; 28 on 4 of 128 in pages of 24, the second 201 / 201 / 167 / 160.  192
//    and 256, whose blocks have an SM to themselves: 8 on 4 of 256 (6, 7, 8, 9, 10), 64 behind 8,192, 1,024 81 / 72 / 71 / 69 / 68, 128 behind 4,096, 2,048
//    188 / 169 / 158 / 158 / 127, 16 on 2, 32 of up to 4 behind 16,000, 300 137 / 149 / 179 / 179 / 179; 10 on 2 of 192 (4, 6, 8, 10), the first 57 / 46 / 48 / 55.
//  * 32 bits, 64 (1, 1.2, 1.5): 14 on 2, 128 behind 4,000, 600 128 / 129 / 120; 8 on 8, the same 143 / 131 / 119; 20 on 1, 256 behind 2,000, 300
//    245 / 208 / 210.
constexpr float kTensorCost = HD <= 64 ? 7.f : 9.f, kPlainCost = HD <= 128 ? 3.5f : HD <= 192 ? 7.f : 9.f, kCost32 = 1.5f;

// `words`: q, its row stride and type, k, v, pages, page, prefix_table and its stride, prefix_lens, groups, prefix limit,
// table and its stride, lengths, requests, limit, cu_groups, cu, out, rows, heads, kv heads, SMs, the rows that a request has
// at most (a hint), scratch and its bytes, err, stream; then the scale as a double.
struct Call {
  own::Args p;
  JoinArgs j;
  FarArgs f;
  int type, longest, groups;
  bool shared, tensor, direct; // tensor: prefixes on the 5th-generation tensor cores
  char* scratch;
  long long room, need;
  cudaStream_t stream;

  explicit Call(const char* words) : p{}, j{}, f{} {
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
    p.sms = num();
    longest = num();
    scratch = (char*)ptr(), room = w[i++];
    p.err = (int*)ptr(), stream = (cudaStream_t)ptr();
    a.scale = (float)*reinterpret_cast<const double*>(w + i);
    a.page_shift = (a.page & (a.page - 1)) == 0 ? 31 - __builtin_clz(a.page) : -1;
    if (longest < 1) longest = 1;
    const bool half = type == GF_BF16;
    groups = half && (long long)longest * (a.nh / a.nkv) > own::kOneGroup ? own::kNearGroups<bf16> : 1;
    const int keys = half ? own::Tile<bf16>::KEYS : own::Tile<float>::KEYS, warps = half ? own::Tile<bf16>::WARPS : own::Tile<float>::WARPS;
    p.rows = 8 * groups;
    p.shape = row_shape_of(a.nh, a.nkv, p.rows);
    p.H = a.nkv * p.shape.chunks;
    const long long item = half ? 2 : 4;
    const bool any = a.G > 0 && a.prefix_limit > 0;
    const long long held = ((any ? a.prefix_limit : 0ll) + a.limit) * HD * item;
    const long long items = (long long)((longest + p.shape.tokens - 1) / p.shape.tokens) * a.B * p.H;
    // (as many of them as there can be: the hint is the longest request's)
    const long long some = ((long long)a.T + (long long)a.B * (p.shape.tokens - 1)) / p.shape.tokens * p.H, reading = items < some ? items : some;
    const long long prefixes = reading * a.prefix_limit * HD * 2 * item;
    p.cluster = 1;
    while (p.cluster < 8 && held > kBlockKeys * (p.cluster > 1 ? p.cluster : 2) && items * p.cluster * 2 <= (p.cluster == 4 ? p.sms * 3 / 4 : p.sms))
      p.cluster *= 2;
    const long long most = p.cluster > 1 && (half || HD <= 64) ? 2 * kDirectKeys : kDirectKeys;
    direct = held <= most * p.cluster && (!any || prefixes <= kDirectBytes) && a.B <= 65535 && p.H <= 65535 &&
             reading <= kDirectWaves * p.sms;
    const long long line = kUnsharedBytes - kUnsharedToken * a.prefix_limit;
    shared = !direct && any && (half || own::kFarGroups > 0) && prefixes > (line > kUnsharedLeast ? line : kUnsharedLeast);
    p.both = !shared, p.joined = !direct, p.after = shared;
    // the scratch: the division, pieces of cut items, of rows, of prefixes
    need = 0;
    auto take = [&](long long bytes) {
      char* here = scratch + need;
      need += (bytes + 255) / 256 * 256;
      return here;
    };
    if (direct) return;
    const long long rows = (long long)a.T * a.nh, cut = (long long)p.sms * warps * 2 * p.rows;
    p.plan = (OwnPlan*)take(16 + (long long)sizeof(OwnPlan::Entry) * a.B);
    p.cut_o = (float*)take(cut * HD * 4), p.cut_ml = (float2*)take(cut * 8);
    if (!shared) return;
    tensor = GF_PREFIX_TC && half && a.page % 8 == 0 && 128 % a.page == 0;
    p.row_o = (float*)take(rows * HD * 4), p.row_ml = (float2*)take(rows * 8);
    j.far_rows = tensor ? 128 : half ? MOST_ROWS : 8 * own::kFarGroups;
    p.far_shape = row_shape_of(a.nh, a.nkv, j.far_rows), p.far_tile = tensor ? 128 : half ? TILE : keys, p.far_H = a.nkv * p.far_shape.chunks;
    p.far_cost = tensor ? kTensorCost : half ? kPlainCost : kCost32;
    const long long tiles = (long long)p.far_H * ((a.T + p.far_shape.tokens - 1) / p.far_shape.tokens + a.G);
    const long long least = 4ll * p.sms * (tensor ? 1 : half ? BLOCKS_AN_SM : warps);
    const long long places = tiles > least ? tiles : least;          // (beyond 2^31 there is no memory for them)
    j.places = (int)(places < INT_MAX ? places : INT_MAX);
    FarPlan* far_plan = (FarPlan*)take((long long)sizeof(FarPlan) * a.G);
    float* far_o = (float*)take(places * j.far_rows * HD * 4);
    float2* far_ml = (float2*)take(places * j.far_rows * 8);
    j.far_plan = far_plan, j.far_o = far_o, j.far_ml = far_ml;
    f = FarArgs{a, 0, p.far_shape, p.shape, p.far_H, p.H, j.places, p.sms, keys, p.far_cost, far_plan, far_o, far_ml, p.err};
  }
};

// The bytes of scratch that a call wants.
GF_EXPORT long long gf_prefix_scratch(const char* words) { return Call(words).need; }

// What gf_prefix_attend returns when it launched one kernel or two; 0: three.
constexpr int kOneLaunch = -101, kTwoLaunches = -102;

template <typename T, int NG, bool FAR>
static int launch_own(const own::Args& p, const CUtensorMap& mk, const CUtensorMap& mv, dim3 grid, cudaStream_t stream) {
  constexpr int threads = 32 * own::Tile<T>::WARPS;
  static OncePerDevice attrs;
  if (int rc = attrs.run([&] {
        return cudaFuncSetAttribute(own::prefix_own_kernel<T, NG, FAR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    (int)own::smem_bytes<T>(NG));
      }))
    return rc;
  if (!p.joined && p.cluster > 1)
    return launch_kernel_cluster_dims(own::prefix_own_kernel<T, NG, FAR>, grid, dim3(threads), own::smem_bytes<T>(NG), stream, p.cluster,
                                      true, mk, mv, p);
  return launch_kernel(own::prefix_own_kernel<T, NG, FAR>, grid, dim3(threads), own::smem_bytes<T>(NG), stream, mk, mv, p);
}
template <typename T>
static int launch_near(const Call& c, const CUtensorMap& mk, const CUtensorMap& mv, dim3 grid) {
  return c.groups == 1 ? launch_own<T, 1, false>(c.p, mk, mv, grid, c.stream)
                       : launch_own<T, own::kNearGroups<T>, false>(c.p, mk, mv, grid, c.stream);
}

GF_EXPORT int gf_prefix_attend(const char* words) {
  Call c(words);
  own::Args& p = c.p;
  PrefixArgs& a = p.a;
  if (a.B <= 0 || a.T <= 0) return 0;
  const bool half = c.type == GF_BF16;
  if (c.need > c.room) return -5;
  // tensor maps: a box is a page's rows of a tile
  auto maps = [&](CUtensorMap& k, CUtensorMap& v, int tile) {
    const int rows = a.page < tile ? a.page : tile;
    return page_map(&k, a.k, a, rows) && page_map(&v, a.v, a, rows);
  };
  auto serves = [&](int tile) { return a.page % 8 == 0 && (tile % a.page == 0 || a.page % tile == 0); };
  CUtensorMap ok{}, ov{};
  p.tma = half && own::Tile<bf16>::SWIZZLED && serves(own::Tile<bf16>::KEYS);
  if (p.tma && !maps(ok, ov, own::Tile<bf16>::KEYS)) return -7;
  if (c.shared) {
    int rc;
#if GF_PREFIX_TC
    if (c.tensor) {
      static OncePerDevice attrs;
      rc = attrs.run([&] {
        return cudaFuncSetAttribute(tc::prefix_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)tc::SMEM);
      });
      if (rc) return rc;
      const FarArgs& f = c.f;
      const tc::Args t{a, f.shape, f.own_shape, f.H, f.own_H, f.places, a.pages * a.page, f.sms, f.own_tile, f.cost, f.far_plan, f.far_o,
                       f.far_ml, f.err};
      CUtensorMap tq, tk, tv;
      if (!query_map(&tq, a, f.shape) || !maps(tk, tv, 128)) return -7;
      rc = launch_kernel(tc::prefix_tc_kernel, dim3(p.sms), dim3(tc::NTHREADS_TC), tc::SMEM, c.stream, tq, tk, tv, t);
    } else
#endif
    if (!half) {
      rc = -6;                   // (no call comes here without kFarGroups: see `shared`)
      if constexpr (own::kFarGroups > 0) {
        own::Args f = p;
        f.shape = p.far_shape, f.H = p.far_H, f.rows = c.j.far_rows, f.own_shape = p.shape, f.own_H = p.H;
        f.places = c.j.places, f.far_plan = c.f.far_plan, f.far_o = c.f.far_o, f.far_ml = c.f.far_ml, f.after = 0;
        rc = launch_own<float, own::kFarGroups, true>(f, ok, ov, dim3(p.sms), c.stream);
      }
    } else {
      static OncePerDevice attrs;
      rc = attrs.run([&] {
        return cudaFuncSetAttribute(prefix_pieces_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PIECES_SMEM);
      });
      if (rc) return rc;
      CUtensorMap fk{}, fv{};
      c.f.tma = SWIZZLED && serves(TILE);
      if (c.f.tma && !maps(fk, fv, TILE)) return -7;
      rc = launch_kernel(prefix_pieces_kernel, dim3(p.sms * BLOCKS_AN_SM), dim3(THREADS), PIECES_SMEM, c.stream, fk, fv, c.f);
    }
    if (rc) return rc;
  }
  const int row_tiles = (c.longest + p.shape.tokens - 1) / p.shape.tokens;
  const dim3 grid = c.direct ? dim3(row_tiles * p.cluster, a.B, p.H) : dim3(p.sms);
  int rc = half ? launch_near<bf16>(c, ok, ov, grid) : launch_near<float>(c, ok, ov, grid);
  if (rc || c.direct) return rc ? rc : kOneLaunch;
  c.j.p = p;
  // (a warp a row where the requests have as many as is said)
  const long long per = (long long)c.longest * (a.nh / a.nkv);
  const unsigned z = (unsigned)(per > 64 * JOIN_WARPS ? 64 : (per + JOIN_WARPS - 1) / JOIN_WARPS);
  rc = launch_kernel(half ? prefix_join_kernel<bf16> : prefix_join_kernel<float>, dim3(a.B, a.nkv, z), dim3(32 * JOIN_WARPS), 0, c.stream,
                     c.j);
  return rc ? rc : c.shared ? 0 : kTwoLaunches;
}
