// The pieces of shared prefixes on the 5th-generation tensor cores, for head sizes 64 and 128 (see shared_prefix.cuh for
// how the work is divided, attention_tc.cu for the same structure over single requests).
//
// A block owns 128 rows, (token, query head) pairs of one kv head, so that a group's requests and their heads share
// every key that is loaded.  Keys come in tiles of 128, which are dealt to two streams; each has its own S, maximum, sum and
// accumulator in tensor memory, and the tensor core works for one while the other's softmax warps turn S into P:
//     S_s = Q K^T (both from shared memory),  P_s in bf16 over S_s's first columns,  O_s += P_s V (P from tensor memory).
// Only a prefix's last tile is masked.  What lies behind its end in its last page may be anything: the weights there are
// zero, and the values are made zero too, since zero times no number is none.
// An item's result is the unnormalised sum of both streams with its maximum and sum, in 32 bits.
//
// What bounds it is a stream's chain of product, softmax and product: with two streams a tile of 128 by 128 takes 1.5 us, 0.55 of
// that its 16,384 exponentials at 16 a clock; the tensor pipe is at work for 44 % of the time, the special-function unit for 46 %.
// Beside own tokens, which have the other SMs: 256 requests behind 32,768 tokens, 40 heads on 8 of 128, 276 us on 123 SMs, 183 tiles each;
// 64 behind 8,192, 28 on 4 of 128, 28 us, 10 of them starts, division and results.
//
// Warps: 0, 1 load K (and Q), 2, 3 load V, 4 issues products, 8 .. 11 and 12 .. 15 are the streams' softmax, a thread a row.
// Every wait on an mbarrier is bounded; when one runs out, an abort flag tells the other roles, all meet at the final barrier
// and tensor memory is freed.
#pragma once
#include "attention_tc.cuh"
#include "shared_prefix.cuh"

namespace gf {
namespace {
namespace tc {

constexpr int QT = 128, KT = 128, NS = 2, HALVES = HD / 64;
constexpr int KS = 2, VS = HD == 128 ? 1 : 2;       // tiles of K and of V a stream
constexpr int NTHREADS_TC = 512, REGS_SMALL = 64, REGS_SOFTMAX = 192;
static_assert(256 * REGS_SMALL + 256 * REGS_SOFTMAX <= 65536, "the register file of an SM");
constexpr uint32_t OPERAND = HALVES * ATOM_BYTES;   // [128 rows][HD]
constexpr uint32_t TMEM_COLS = 512;                 // S_0 / P_0: 0..127, S_1 / P_1: 128..255, O_0, O_1: 256..
constexpr float kRescaleStep = 8.f;                 // log2 units a maximum may grow before O is rescaled
constexpr int kOver = 2;                            // what an item costs beside its tiles

struct Barriers {
  uint64_t q_full, q_empty;
  uint64_t k_full[NS * KS], k_empty[NS * KS], v_full[NS * VS], v_empty[NS * VS];
  uint64_t s_full[NS], p_ready[NS], pv_done[NS], stat_ready, o_free, drained;
  uint32_t tmem_base;
  int abort_flag, chunk, workers;
  GroupTiles groups[32];       // the first 32 groups'
  long long own[8];
  float stat_m[NS][QT], stat_l[NS][QT];
};
constexpr uint32_t SMEM = OPERAND * (1 + NS * KS + NS * VS) + sizeof(Barriers);

struct Args {
  PrefixArgs a;
  Shape shape, own_shape;      // rows of this kernel's tiles, of the one's that works on own tokens beside it
  int H, own_H, places, oob_row, sms, own_tile;
  float cost;                  // of a tile beside one of own tokens
  FarPlan* far_plan;           // [G]
  float* far_o;                // [places][QT][HD]
  float2* far_ml;
  int* err;
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// Weights are summed as they are rounded for the product, as in the other kernels: a row that one key takes nearly all of gets
// its value as it is.  (Summed as they come, in packed additions, the kernel is 2 to 5 % faster and such rows are off by a step of
// bfloat16; unpacked by integer instructions first, 3 to 8 % slower than that.)
__device__ __forceinline__ void add_rounded(float& a, float& b, uint32_t pair) {
  uint16_t lo, hi;
  asm("mov.b32 {%0, %1}, %2;" : "=h"(lo), "=h"(hi) : "r"(pair));
  asm("add.rn.f32.bf16 %0, %1, %0;" : "+f"(a) : "h"(lo));
  asm("add.rn.f32.bf16 %0, %1, %0;" : "+f"(b) : "h"(hi));
}

__global__ void __launch_bounds__(NTHREADS_TC, 1)
prefix_tc_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                 const __grid_constant__ CUtensorMap tmap_v, const Args g) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* q_s = smem_raw;                           // (no static shared memory: the tiles start at the aligned base)
  unsigned char* k_s = q_s + OPERAND;
  unsigned char* v_s = k_s + NS * KS * OPERAND;
  Barriers* bars = reinterpret_cast<Barriers*>(v_s + NS * VS * OPERAND);
  volatile int* abort_flag = &bars->abort_flag;
  const PrefixArgs& a = g.a;
  int* err = g.err;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int box_rows = g.shape.tokens * g.shape.heads;     // rows of Q that come by TMA
  pdl_wait();
  pdl_trigger();               // (behind the wait: the kernel beside this one reads what was waited for)
  if (smem_u32(smem_raw) & 1023u) {
    if (threadIdx.x == 0 && err) atomicExch(err, 31);
    return;
  }
  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    mbar_init(&bars->q_empty, 1);
    for (int s = 0; s < NS * KS; ++s) {
      mbar_init(&bars->k_full[s], 2);          // one arrival (with its byte count) per loader warp
      mbar_init(&bars->k_empty[s], 1);
    }
    for (int s = 0; s < NS * VS; ++s) {
      mbar_init(&bars->v_full[s], 2);
      mbar_init(&bars->v_empty[s], 1);
    }
    for (int s = 0; s < NS; ++s) {
      mbar_init(&bars->s_full[s], 1);
      mbar_init(&bars->p_ready[s], QT);
      mbar_init(&bars->pv_done[s], 1);
    }
    mbar_init(&bars->stat_ready, NS * QT);
    mbar_init(&bars->o_free, NS * QT);
    mbar_init(&bars->drained, 1);
    bars->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&bars->tmem_base)), "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // how the prefixes and the own tokens share the SMs: own tokens counted by the first eight warps
  GroupTiles t{};
  FarWork f{};
  if (warp == 5) f = far_work(a, t, g.H, g.shape.tokens, KT);
  const OwnWork own = own_work<256>(a, g.own_shape.tokens, g.own_tile, false, bars->own);
  if (warp == 5) {
    const int workers = min((int)gridDim.x, far_share(g.sms, f.priced, g.cost, own.total * g.own_H));
    const int chunk = plan_chunk(a, t, f, g.H, g.shape.tokens, KT, max(workers, 1), g.places, kOver);
    bars->groups[lane] = t;
    if (lane == 0) {
      bars->chunk = chunk, bars->workers = workers;
    }
    if (blockIdx.x == 0) write_far_plan(a, t, g.H, g.shape.tokens, KT, chunk, g.far_plan);
  }
  // rows that no token fills are zeros, so that their scores are numbers
  for (int i = box_rows * 8 + threadIdx.x; i < QT * 8; i += NTHREADS_TC)
    for (int h = 0; h < HALVES; ++h) reinterpret_cast<uint4*>(q_s + h * ATOM_BYTES)[i] = make_uint4(0u, 0u, 0u, 0u);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = bars->tmem_base, tmem_s = tmem, tmem_o = tmem + NS * KT;
  const int chunk = bars->chunk, workers = bars->workers;
  const GroupTiles groups = bars->groups[lane];
  PrefixItem it;
  // the block's n-th item; by whole warps
  auto item_of = [&](int n) {
    const int index = n * workers + (int)blockIdx.x;
    return (int)blockIdx.x < workers && index < g.places && find_item(a, groups, g.H, g.shape.tokens, KT, chunk, index, it);
  };
  auto tiles_of = [](int ntiles, int s) { return (ntiles - s + 1) >> 1; };     // of stream s

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_SMALL));
    // ------------------------------------------------------------------ loaders: every other box of K (0, 1) or V (2, 3)
    const bool is_v = warp >= 2;
    const int part = warp & 1, page_size = a.page;
    const int ops = KT / page_size * HALVES, my_ops = (ops - part + 1) / 2;
    constexpr int MAX_OPS = ((KT / 8) * HALVES / 2 + 31) / 32;                 // page sizes down to 8
    const int per_stream = is_v ? VS : KS;
    unsigned char* ring = is_v ? v_s : k_s;
    uint64_t* full = is_v ? bars->v_full : bars->k_full;
    uint64_t* empty = is_v ? bars->v_empty : bars->k_empty;
    const CUtensorMap* map = is_v ? &tmap_v : &tmap_k;
    const uint32_t my_bytes = (uint32_t)my_ops * (uint32_t)page_size * 128u;
    int cs[NS] = {0, 0}, seq = 0;
    bool go = true;
    for (int n = 0; go && item_of(n); ++n) {
      const int* tbl = a.prefix_table + (size_t)it.g * a.prefix_stride;
      const int j0 = it.split * chunk, ntiles = min(chunk, it.tiles - j0), end = it.length;
      const int kvh = it.hc / g.shape.chunks, kv_col = kvh * HD;
      if (warp == 0) {
        int ok = 1;
        if (lane == 0) {
          ok = mbar_wait(&bars->q_empty, (uint32_t)(seq & 1) ^ 1u, abort_flag, err, 32);
          if (ok) {
            mbar_expect_tx(&bars->q_full, (uint32_t)HALVES * box_rows * 128u);
            for (int h = 0; h < HALVES; ++h)
              tma_load_3d(q_s + h * ATOM_BYTES, &tmap_q, &bars->q_full, h * 64,
                          kvh * (a.nh / a.nkv) + (it.hc - kvh * g.shape.chunks) * g.shape.heads, it.first);
            ++seq;
          }
        }
        if (!__shfl_sync(0xffffffffu, ok, 0)) { go = false; break; }
      }
      int rows_next[MAX_OPS];
      auto lookup = [&](int i) {
        const int key0 = (j0 + i) * KT;
#pragma unroll
        for (int u = 0; u < MAX_OPS; ++u) {
          const int op = part + 2 * (lane + 32 * u);
          rows_next[u] = g.oob_row;                  // pages behind the prefix: TMA fills them with zeros
          if (op < ops && i < ntiles) {
            const int c = key0 + (op / HALVES) * page_size;
            if (c < end) rows_next[u] = page_in(a, fresh_index(tbl + logical_page(a, c))) * page_size;
          }
        }
      };
      lookup(0);
      for (int i = 0; i < ntiles; ++i) {
        int rows_now[MAX_OPS];
#pragma unroll
        for (int u = 0; u < MAX_OPS; ++u) rows_now[u] = rows_next[u];
        int& cnt = (i & 1) ? cs[1] : cs[0];
        const int st = (i & 1) * per_stream + cnt % per_stream;
        int ok = 1;
        if (lane == 0) {
          ok = mbar_wait(&empty[st], ((cnt / per_stream) & 1) ^ 1, abort_flag, err, 33);
          if (ok && my_bytes) mbar_expect_tx(&full[st], my_bytes);
          else if (ok) mbar_arrive(&full[st]);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) { go = false; break; }
#pragma unroll
        for (int u = 0; u < MAX_OPS; ++u) {
          const int op = part + 2 * (lane + 32 * u);
          if (op < ops) {
            const int pg = op / HALVES, h = op - pg * HALVES;
            tma_load_2d(ring + (size_t)st * OPERAND + h * ATOM_BYTES + (size_t)pg * page_size * 128, map, &full[st],
                        kv_col + h * 64, rows_now[u]);
          }
        }
        ++cnt;
        lookup(i + 1);
      }
    }
    // (a wait that ran out: nothing may still be on its way into this block's memory when it ends)
    if (!go && lane == 0) {
      if (warp == 0 && seq > 0) wait_bar(&bars->q_full, (uint32_t)(seq - 1) & 1u, err, 43);
      for (int s = 0; s < NS; ++s)
        for (int c = max(0, cs[s] - per_stream); c < cs[s]; ++c)
          wait_bar(&full[s * per_stream + c % per_stream], (uint32_t)(c / per_stream) & 1u, err, 43);
    }
    __syncwarp();
  } else if (warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_SMALL));
    // ------------------------------------------------------------------ products: P V and the next S of stream 0, then of 1
    if (warp == 4) {
      constexpr uint32_t id_qk = idesc(KT, false), id_pv = idesc(HD, true);
      const uint32_t q_desc = desc_lo_kmajor(smem_u32(q_s)), k_desc = desc_lo_kmajor(smem_u32(k_s)),
                     v_desc = desc_lo_mnmajor(smem_u32(v_s));
      int seq = 0, ck0 = 0, ck1 = 0, cv0 = 0, cv1 = 0;
      bool ok = true;
      for (int n = 0; ok && item_of(n); ++n) {
        const int ntiles = min(chunk, it.tiles - it.split * chunk);
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->q_full, (uint32_t)(seq & 1), abort_flag, err, 34));
        auto issue_qk = [&](int s, bool last) {
          int& ck = s ? ck1 : ck0;
          const int st = s * KS + ck % KS;
          if (lane == 0) {
            const uint32_t kd = k_desc + st * (OPERAND >> 4);
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
              const uint32_t off = ((k / 4) * ATOM_BYTES + (k % 4) * 32) >> 4;
              umma(tmem_s + KT * s, make_desc(q_desc + off), make_desc(kd + off), id_qk, k > 0 ? 1u : 0u);
            }
            umma_commit(&bars->s_full[s]);
            if (last) umma_commit(&bars->q_empty);
          }
          ++ck;
        };
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          if (s >= ntiles || !ok) continue;
          const int ck = s ? ck1 : ck0;
          ok = __all_sync(0xffffffffu, mbar_wait<true>(&bars->k_full[s * KS + ck % KS], (ck / KS) & 1, abort_flag, err, 35));
          if (!ok) continue;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          issue_qk(s, s == ntiles - 1);
        }
        const int n0 = tiles_of(ntiles, 0);
        for (int t = 0; t < n0 && ok; ++t) {
#pragma unroll
          for (int s = 0; s < NS; ++s) {
            const int i = NS * t + s;
            if (i >= ntiles || !ok) continue;
            int& cv = s ? cv1 : cv0;
            const int ck = s ? ck1 : ck0, st = s * VS + cv % VS;
            // the item's first P V overwrites O: the item before must have been read out
            if (i == 0)
              ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_free, (uint32_t)(seq & 1) ^ 1u, abort_flag, err, 36));
            // lane 0: P of this tile; lane 1: its V tile; lane 2: the K tile of the next S product
            {
              uint64_t* bar = lane == 0 ? &bars->p_ready[s] : lane == 1 ? &bars->v_full[st] : &bars->k_full[s * KS + ck % KS];
              const uint32_t par = lane == 0 ? (cv & 1) : lane == 1 ? ((cv / VS) & 1) : ((ck / KS) & 1);
              const bool active = lane < 2 || (lane == 2 && i + NS < ntiles);
              if (ok) ok = mbar_wait_lanes(bar, par, active, abort_flag, err, 37);
            }
            if (!ok) continue;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (lane == 0) {
              const uint32_t vd = v_desc + st * (OPERAND >> 4);
#pragma unroll
              for (int k = 0; k < KT / 16; ++k)      // 16 keys: 8 columns of P, 16 rows of V
                umma_ts(tmem_o + HD * s, tmem_s + KT * s + 8 * k, make_desc(vd + ((k * 16 * 128) >> 4)), id_pv,
                        (t > 0 || k > 0) ? 1u : 0u);
            }
            if (i + NS < ntiles) issue_qk(s, i + NS == ntiles - 1);
            if (lane == 0) {
              umma_commit(&bars->v_empty[st]);
              if (i + NS >= ntiles) umma_commit(&bars->pv_done[s]);
            }
            ++cv;
          }
        }
        ++seq;
      }
      if (!ok) {                   // (likewise: products under way end before tensor memory is given back)
        if (lane == 0) {
          umma_commit(&bars->drained);
          wait_bar(&bars->drained, 0u, err, 44);
        }
        __syncwarp();
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    // ------------------------------------------------------------------ softmax and results (a wait's end is the warp's)
    const int qd = warp & 3, s = (warp - 8) >> 2, r = qd * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(qd * 32) << 16;
    const uint32_t my_s = tmem_s + KT * s + lane_addr, my_o = tmem_o + HD * s + lane_addr;
    const float scale_log2 = a.scale * LOG2E;
    int cnt = 0, seq = 0, had = 0;
    bool ok = true;
    for (int n = 0; ok && item_of(n); ++n) {
      const int j0 = it.split * chunk, ntiles = min(chunk, it.tiles - j0), mine = tiles_of(ntiles, s), end = it.length;
      const bool live = r < it.count * g.shape.heads;
      float m_used = -INFINITY, l = 0.f;
      for (int t = 0; t < mine; ++t, ++cnt) {
        ok = __all_sync(0xffffffffu, mbar_wait<true>(&bars->s_full[s], cnt & 1, abort_flag, err, 38));
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (r == 0) mbar_arrive(&bars->k_empty[s * KS + cnt % KS]);   // S is computed: its K tile is free
        __syncwarp();                  // (tensor memory's instructions want the warp as one)
        const int left = end - (j0 + 2 * t + s) * KT;                 // keys of the tile that are the prefix's
        float v[KT];
#pragma unroll
        for (int cc = 0; cc < KT / 32; ++cc) tmem_ld32(my_s + 32 * cc, *reinterpret_cast<float(*)[32]>(v + 32 * cc));
        tmem_ld_wait();
        if (left < KT) {
#pragma unroll
          for (int k = 0; k < KT; ++k) v[k] = k < left ? v[k] : -INFINITY;
          // the prefix's last tile: values behind its end become zeros
          const int st = s * VS + cnt % VS;
          ok = __all_sync(0xffffffffu, mbar_wait<true>(&bars->v_full[st], (cnt / VS) & 1, abort_flag, err, 39));
          if (!ok) break;
          if (r >= left)
            for (int h = 0; h < HALVES; ++h)
#pragma unroll
              for (int c = 0; c < 8; ++c)
                reinterpret_cast<uint4*>(v_s + (size_t)st * OPERAND + h * ATOM_BYTES + r * 128)[c] = make_uint4(0u, 0u, 0u, 0u);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        float mx8[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) mx8[j] = -INFINITY;
#pragma unroll
        for (int k = 0; k < KT; k += 2) mx8[(k >> 1) & 7] = max3(mx8[(k >> 1) & 7], v[k], v[k + 1]);
        const float mx = fmaxf(max3(mx8[0], mx8[1], mx8[2]), max3(mx8[3], mx8[4], max3(mx8[5], mx8[6], mx8[7]))) * scale_log2;
        // the old maximum is kept unless the row's outgrew it
        float m_new = m_used;
        if (mx > m_used + kRescaleStep || m_used == -INFINITY) m_new = fmaxf(m_used, mx);
        const float corr = (m_new == m_used) ? 1.f : (m_used == -INFINITY ? 0.f : fast_exp2(m_used - m_new));
        const float msub = m_new == -INFINITY ? 0.f : m_new;
        // (S of this tile is complete, so the stream's P V of the tile before is too: O_s is at rest)
        if (t > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll 1
          for (int cc = 0; cc < HD; cc += 16) {
            float o[16];
            tmem_ld16(my_o + cc, o);
            tmem_ld_wait();
            uint32_t ob[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) ob[k] = __float_as_uint(o[k] * corr);
            tmem_st16(my_o + cc, ob);
          }
        }
        float sum[4] = {};
        const uint64_t scale2 = pack2(scale_log2, scale_log2), msub2 = pack2(-msub, -msub);
#pragma unroll
        for (int cc = 0; cc < KT / 32; ++cc) {
          uint32_t w[16];
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float a0, a1;
            unpack2(fma2(pack2(v[32 * cc + k], v[32 * cc + k + 1]), scale2, msub2), a0, a1);
            w[k / 2] = pack_bf16(fast_exp2(a0), fast_exp2(a1));
            add_rounded(sum[k & 2], sum[(k & 2) + 1], w[k / 2]);
          }
          tmem_st16(my_s + 16 * cc, w);
        }
        l = l * corr + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
        m_used = m_new;
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        mbar_arrive(&bars->p_ready[s]);
      }
      if (!ok) break;
      if (mine > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->pv_done[s], had & 1, abort_flag, err, 40));
        ++had;
      }
      if (!ok) break;
      // (the item before has been read out by every thread, so its figures are not needed any more)
      if (seq > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars->o_free, (uint32_t)(seq - 1) & 1u, abort_flag, err, 41));
      if (!ok) break;
      bars->stat_m[s][r] = m_used;
      bars->stat_l[s][r] = l;
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      mbar_arrive(&bars->stat_ready);
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->stat_ready, seq & 1, abort_flag, err, 42));
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const float m_o = bars->stat_m[s ^ 1][r], l_o = bars->stat_l[s ^ 1][r];
      const float m_all = fmaxf(m_used, m_o);
      const float f_me = m_used == -INFINITY ? 0.f : fast_exp2(m_used - m_all);
      const float f_o = m_o == -INFINITY ? 0.f : fast_exp2(m_o - m_all);
      const float f0 = s == 0 ? f_me : f_o, f1 = s == 0 ? f_o : f_me;
      const bool two = ntiles > 1;
      const uint32_t o0 = tmem_o + lane_addr + s * (HD / 2), o1 = o0 + HD;
      const size_t at = (size_t)(n * workers + (int)blockIdx.x) * QT + r;
      float* to = g.far_o + at * HD + s * (HD / 2);
      if (live && s == 0) g.far_ml[at] = make_float2(m_all, l * f_me + l_o * f_o);
#pragma unroll 1
      for (int cc = 0; cc < HD / 2; cc += 16) {
        float x[16], y[16];
        __syncwarp();
        tmem_ld16(o0 + cc, x);
        if (two) tmem_ld16(o1 + cc, y);
        tmem_ld_wait();
        if (cc + 16 >= HD / 2) {
          // O is read: the next item's first P V may overwrite it while this one is stored
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          mbar_arrive(&bars->o_free);
        }
        if (live) {
#pragma unroll
          for (int k = 0; k < 16; ++k) x[k] = two ? fmaf(y[k], f1, x[k] * f0) : x[k] * f0;
#pragma unroll
          for (int k = 0; k < 16; k += 8)            // (a whole sector a thread)
            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + cc + k), "f"(x[k]), "f"(x[k + 1]),
                         "f"(x[k + 2]), "f"(x[k + 3]), "f"(x[k + 4]), "f"(x[k + 5]), "f"(x[k + 6]), "f"(x[k + 7])
                         : "memory");
        }
      }
      ++seq;
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 4) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
}

}  // namespace tc
}  // namespace
}  // namespace gf
